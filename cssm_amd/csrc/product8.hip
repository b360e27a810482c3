// Matrix product of 8-bit rows and an 8-bit weight (gfx950):
//   out[m][n] = act(sum over 128-blocks b of 2^(sa[m][b] + sw[n / 128][b]) sum_{k in b} a[m][k] w[n][k] + bias[n])
// a (M, K), w (N, K) e4m3.  Two forms, by the output's type:
//   bfloat16  the 8-bit matrix instruction.  The scales are powers of two, which its scaled form applies exactly in the
//             float32 accumulation.  It takes one for each 32 of k; all of a block's get the same byte, so the order of k
//             within a block does not matter as long as both sides agree.  The instruction adds the products of
//             neighbouring k with what lies about 13 bits below the largest of them dropped: 1.4e-5 of a result of
//             normal values, 1 / 100 of the output's own rounding.
//   float32   the values as bfloat16, which holds each exactly, on the bfloat16 instruction, whose sums are off by a
//             float32 rounding (1e-8 .. 1e-7 measured), each block's sum scaled as it joins the others.
// The weight is the instruction's first operand: a lane then holds four consecutive n of one m.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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

// ---- many rows: tiles through LDS
// A workgroup takes BM rows x BN columns of the output, in steps of one 128-block of k.  Each step's rows (128 bytes each)
// go from memory to LDS without passing registers, one step ahead of the products; the 16-byte pieces of a row are
// stored at piece ^ (row % 8), so that the 8 lanes that LDS serves at once, 8 rows at the same piece, meet 8 different
// bank groups.  256 x 256 on 8 waves (128 x 64 each): 192 KB of LDS reads a step against 2061 cycles of products, 75 % of
// what LDS gives; a smaller tile's waves would wait for LDS instead.
// Bound by the matrix cores where the tiles fill the chip: 8192 x 8192 x 4096 to bf16 277 us, 1.98 PFLOP/s (the median of 100
// in a row; 270 to 310 with other pauses between them, as the clock goes); to float32 630 us, 0.87 (the bf16 instruction
// has half the 8-bit one's rate, and every row fragment is widened for each of the wave's two column tiles).  128 x 128 tiles
// where the large ones would leave a quarter of the CUs without one; they do not split K, so that few of them cannot fill the
// chip: 256 x 4096 x 4096 28 us, 1024 x 4096 x 4096 33.

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// 16 bytes a lane from base + offset to LDS at `to` + 16 lane (to: the same for the wave).  No vector register is written;
// the wait is wait_copies().  The place goes by way of m0, which a clobber list cannot name: it is handed back as it was.
__device__ __forceinline__ void copy_to_lds(const uint8_t* base, uint32_t offset, uint32_t to) {
  uint32_t was;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
               : "=&s"(was) : "s"(to), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Output tile of workgroup `id`: workgroups go round the 8 XCDs, so each XCD gets a run of tiles, and a run walks bands
// of 8 row tiles column by column: the 32 tiles that an XCD works on share 8 rows' and 4 columns' operands in its L2.
__device__ __forceinline__ void tile_of(int id, int nmt, int nnt, int& mt, int& nt) {
  const int n = nmt * nnt, x = id % 8, q = n / 8, r = n % 8;
  const int t = x * q + min(x, r) + id / 8;
  const int band = t / (8 * nnt), rows = min(8, nmt - band * 8), in = t - band * 8 * nnt;
  mt = band * 8 + in % rows;
  nt = in / rows;
}

template <typename O>
struct Whole {
  O v[16 / sizeof(O)];
};

template <int BM, int BN, int WM, int WN, typename O, bool WIDE>
__global__ void __launch_bounds__(WM* WN * 64) product_tiles(Product8 p) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, PIECES = (BM + BN) / 8 / WAVES;
  static_assert(BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0 && 128 % (TN * 32) == 0, "");
  constexpr int SCALES = 64;   // steps whose exponents lie in LDS at a time
  __shared__ uint4 lds[2][(BM + BN) * 8];
  __shared__ uint8_t sa[SCALES][BM];
  __shared__ uint8_t sw[SCALES][BN < 128 ? 1 : BN / 128];
  int mt, nt;
  tile_of(int(blockIdx.x), (p.M + BM - 1) / BM, (p.N + BN - 1) / BN, mt, nt);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x % 64;
  const int m0 = mt * BM, n0 = nt * BN, nw = n0 + wave / WM * (TN * 32);
  const int nkb = (p.K + 127) / 128, whole = p.K / 128;
  const uint8_t* ab = p.a + size_t(m0) * p.K;
  const uint8_t* wb = p.w + size_t(n0) * p.K;
  // The wave copies pieces of 8 rows each step, number wave, wave + WAVES, ..: first a's, then w's.  (The row is hidden from
  // the compiler, which would keep every piece's address in a register through the loop.)
  const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>(&lds[0][0]));
  int myrow = wave * 8 + l / 8;
  const uint32_t mypart = uint32_t((l % 8 ^ l / 8) * 16);
  auto from = [&](int i) {
    const int row = i * WAVES * 8 + myrow;
    const int r = i * WAVES * 8 < BM ? min(row, p.M - 1 - m0) : min(row - BM, p.N - 1 - n0);
    return uint32_t(r) * uint32_t(p.K) + mypart;
  };
  auto fetch = [&](int b) {
    asm volatile("" : "+v"(myrow));
    if (b < whole) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        copy_to_lds((i * WAVES * 8 < BM ? ab : wb) + size_t(b) * 128, from(i),
                    lds0 + uint32_t((b & 1) * sizeof(lds[0]) + (i * WAVES + wave) * 1024));
    } else {   // the last block of a K between multiples of 128: zeros behind it (K is a multiple of 16)
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (b * 128 + int(mypart) < p.K) v = *reinterpret_cast<const uint4*>((i * WAVES * 8 < BM ? ab : wb) + size_t(b) * 128 + from(i));
        lds[b & 1][(i * WAVES + wave) * 64 + l] = v;
      }
    }
  };
  auto fetch_scales = [&](int b0) {
    const int n = min(SCALES, nkb - b0);
    for (int row = threadIdx.x; row < BM; row += WAVES * 64) {
      const uint8_t* s = p.sa + size_t(min(m0 + row, p.M - 1)) * nkb + b0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) sa[i][row] = s[i];
    }
    for (int i = threadIdx.x; i < n * (BN / 128); i += WAVES * 64)
      sw[i / (BN / 128)][i % (BN / 128)] = p.sw[size_t(min(n0 / 128 + i % (BN / 128), (p.N - 1) / 128)) * nkb + b0 + i / (BN / 128)];
  };
  f32x16_t acc[TN][TM] = {};
  // piece c of the lane's row in row tile t of a (0) or w (BM / 32)
  auto piece = [&](const uint4* s, int t, int c) { return s[(t * 32 + l % 32) * 8 + (c ^ l % 8)]; };
  auto frag = [&](const uint4* s, int t, int c) {
    const uint4 lo = piece(s, t, c), hi = piece(s, t, c + 1);
    return i32x8_t{int(lo.x), int(lo.y), int(lo.z), int(lo.w), int(hi.x), int(hi.y), int(hi.z), int(hi.w)};
  };
  auto step = [&](int b) {
    const uint4* s = lds[b & 1];
    const int ta = wave % WM * TM, tw = BM / 32 + wave / WM * TN;
    int ea[TM];
    const int ew = sw[b % SCALES][(nw - n0) / 128];
#pragma unroll
    for (int j = 0; j < TM; ++j) ea[j] = sa[b % SCALES][(ta + j) * 32 + l % 32];
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        bf16x8_t fw[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 q = piece(s, tw + i, c * 2 + l / 32);
          fw[2 * c] = widen(int(q.x), int(q.y)), fw[2 * c + 1] = widen(int(q.z), int(q.w));
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          asm volatile("" ::: "memory");
          f32x16_t part = {};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint4 q = piece(s, ta + j, c * 2 + l / 32);
            part = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fw[2 * c], widen(int(q.x), int(q.y)), part, 0, 0, 0);
            part = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fw[2 * c + 1], widen(int(q.z), int(q.w)), part, 0, 0, 0);
          }
          const int e = ew + ea[j] - 254;
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[i][j][v] += __builtin_amdgcn_ldexpf(part[v], e);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        i32x8_t fw[TN];
#pragma unroll
        for (int i = 0; i < TN; ++i) fw[i] = frag(s, tw + i, h * 4 + l / 32 * 2);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const i32x8_t fa = frag(s, ta + j, h * 4 + l / 32 * 2);
#pragma unroll
          for (int i = 0; i < TN; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[i], fa, acc[i][j], 0, 0, 0, ew, 0, ea[j]);
        }
      }
    }
  };
  fetch(0);
  for (int b = 0; b < nkb; ++b) {
    if (b % SCALES == 0) {
      __syncthreads();
      fetch_scales(b);
    }
    wait_copies();
    __syncthreads();   // step b's rows are there, and everyone is done with the step before it, whose place b + 1 takes
    if (b + 1 < nkb) fetch(b + 1);
    step(b);
  }
  // To memory by way of LDS, 32 rows of each wave at a time, so that whole lines are written: a lane holds 4 columns of a
  // row, 32 lanes 32 rows.  The 16-byte pieces of a row lie at piece ^ row, which spreads both ways over the banks.
  constexpr int LINE = BN * int(sizeof(O)) / 16, ROWS = WM * 32, HALF = LINE * ROWS;   // pieces of a row, rows and pieces of a turn
  constexpr bool TWICE = 2 * HALF <= 2 * (BM + BN) * 8;   // room for two turns: one barrier each
  uint4* buf = &lds[0][0];
  const bool whole16 = p.N % (16 / int(sizeof(O))) == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  auto write_out = [&](auto act) {
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      uint4* to = buf + (TWICE ? (j & 1) * HALF : 0);
      if (j == 0 || !TWICE) __syncthreads();   // the products, or the turn before, are done with LDS
      const int row = wave % WM * 32 + l % 32;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = nw - n0 + i * 32 + e * 8 + l / 32 * 4, n = n0 + col;
          float o[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = activate(acc[i][j][e * 4 + v] + (p.bias ? p.bias[min(n + v, p.N - 1)] : 0.0f), decltype(act)::value);
          const int at = col * int(sizeof(O));
          store_row<4>(reinterpret_cast<O*>(reinterpret_cast<uint8_t*>(to + row * LINE + (at / 16 ^ row % LINE)) + at % 16), o);
        }
      __syncthreads();   // (the turn before last has been read by then)
      for (int k = threadIdx.x; k < HALF; k += WAVES * 64) {
        const int r = k / LINE, c = k % LINE, m = m0 + r / 32 * (TM * 32) + j * 32 + r % 32;
        const int n = n0 + c * (16 / int(sizeof(O)));
        if (m >= p.M || n >= p.N) continue;
        const uint4 q = to[r * LINE + (c ^ r % LINE)];
        O* out = static_cast<O*>(p.out) + size_t(m) * p.N + n;
        if (whole16) {
          *reinterpret_cast<uint4*>(out) = q;
        } else {
#pragma unroll
          for (int v = 0; v < 16 / int(sizeof(O)); ++v)
            if (n + v < p.N) out[v] = __builtin_bit_cast(Whole<O>, q).v[v];
        }
      }
    }
  };
  if (p.act == 1) write_out(std::integral_constant<int, 1>());
  else if (p.act == 2) write_out(std::integral_constant<int, 2>());
  else write_out(std::integral_constant<int, 0>());
}

// ---- few rows: the weight streams past
// 16 TN columns a workgroup, the blocks of k dealt to its waves, whose sums meet in LDS in order.  A wave reads whole
// lines of the weight, AHEAD blocks at a time, and the rows (few: L2 holds them) beside.  Bound by the weight's bytes; from
// 17 rows on, and where N gives every CU a workgroup, 32 columns halve what the rows cost (16 x 8192 x 4096 11.9 -> 9.6
// us on the same operands each time, 11 on others in turn; 16 x 1024 x 1024 the other way, 4.0 -> 7.0).  Each workgroup reads
// all rows again, which counts from 32 rows on: 32 x 8192 x 4096 13.6 us, 64 x 8192 x 4096 20.

// 32 bytes at base + offset, zeros behind the `left` that there are of the row (a multiple of 16)
__device__ __forceinline__ i32x8_t load32(const uint8_t* base, uint32_t offset, int left) {
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (left > 0) lo = *reinterpret_cast<const uint4*>(base + offset);
  if (left > 16) hi = *reinterpret_cast<const uint4*>(base + offset + 16);
  return i32x8_t{int(lo.x), int(lo.y), int(lo.z), int(lo.w), int(hi.x), int(hi.y), int(hi.z), int(hi.w)};
}

template <int TM, int TN, int WAVES, int AHEAD, typename O, bool WIDE>
__global__ void __launch_bounds__(WAVES * 64) product_rows(Product8 p) {
  __shared__ float sums[WAVES][TN][TM][4][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x % 64, r = l % 16, kq = l / 16;
  const int n0 = int(blockIdx.x) * (16 * TN), m0 = int(blockIdx.y) * (16 * TM), nkb = (p.K + 127) / 128;
  const uint8_t* ab = p.a + size_t(m0) * p.K;
  const uint8_t* sb = p.sa + size_t(m0) * nkb;
  const uint8_t* wb = p.w + size_t(n0) * p.K;
  const uint8_t* ws = p.sw + size_t(n0 / 128) * nkb;
  uint32_t wr[TN], ar[TM], as[TM];   // (at most 64 rows of fewer than 2^24 bytes)
#pragma unroll
  for (int i = 0; i < TN; ++i) wr[i] = uint32_t(min(i * 16 + r, p.N - 1 - n0)) * uint32_t(p.K) + uint32_t(kq * 32);
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const uint32_t m = uint32_t(min(j * 16 + r, p.M - 1 - m0));
    ar[j] = m * uint32_t(p.K) + uint32_t(kq * 32);
    as[j] = m * uint32_t(nkb);
  }
  f32x4_t acc[TN][TM] = {};
  for (int b0 = wave; b0 < nkb; b0 += WAVES * AHEAD) {
    i32x8_t fw[AHEAD][TN], fa[AHEAD][TM];
    int sw[AHEAD], sa[AHEAD][TM];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int b = b0 + WAVES * u, k = b * 128 + kq * 32;
      if (b >= nkb) continue;
#pragma unroll
      for (int i = 0; i < TN; ++i) fw[u][i] = load32(wb + size_t(b) * 128, wr[i], p.K - k);
      sw[u] = ws[b];
#pragma unroll
      for (int j = 0; j < TM; ++j) fa[u][j] = load32(ab + size_t(b) * 128, ar[j], p.K - k), sa[u][j] = (sb + b)[as[j]];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (b0 + WAVES * u >= nkb) continue;
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          if constexpr (WIDE) {
            f32x4_t part = {};
#pragma unroll
            for (int s = 0; s < 4; ++s)
              part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(fw[u][i][2 * s], fw[u][i][2 * s + 1]),
                                                             widen(fa[u][j][2 * s], fa[u][j][2 * s + 1]), part, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] += __builtin_amdgcn_ldexpf(part[e], sw[u] + sa[u][j] - 254);
          } else {
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u][i], fa[u][j], acc[i][j], 0, 0, 0, sw[u], 0, sa[u][j]);
          }
        }
    }
  }
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[wave][i][j][e][l] = acc[i][j][e];
  __syncthreads();
  const bool wide = p.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % (4 * sizeof(O)) == 0;
  for (int t = wave; t < TN * TM; t += WAVES) {
    const int i = t / TM, j = t % TM, m = m0 + j * 16 + r, n = n0 + i * 16 + kq * 4;
    if (m >= p.M || n >= p.N) continue;
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += sums[w][i][j][e][l];
      o[e] = activate(s + (p.bias && n + e < p.N ? p.bias[n + e] : 0.0f), p.act);
    }
    store4(static_cast<O*>(p.out), size_t(m) * p.N + n, n, p.N, wide, o);
  }
}

template <typename O, bool WIDE>
void launch(const Product8& p, hipStream_t s) {
  const auto over = [](int n, int d) { return unsigned((n + d - 1) / d); };
  // up to 128 rows this way where the tiles would leave most CUs without one (128 x 4096 x 4096, 32 tiles: 25 us, this way 19)
  if (p.M <= 64 || (p.M <= 128 && over(p.N, 128) < 64)) {
    if (p.M <= 16 && p.N < 8192) product_rows<1, 1, 4, 4, O, WIDE><<<over(p.N, 16), 256, 0, s>>>(p);
    else if (p.M <= 16) product_rows<1, 2, 8, 4, O, WIDE><<<over(p.N, 32), 512, 0, s>>>(p);
    else if (p.M <= 32) product_rows<2, 2, 8, 2, O, WIDE><<<over(p.N, 32), 512, 0, s>>>(p);
    else product_rows<4, 2, 8, 2, O, WIDE><<<dim3(over(p.N, 32), over(p.M, 64)), 512, 0, s>>>(p);
  } else if (over(p.M, 256) * over(p.N, 256) >= 192) {
    if constexpr (WIDE) product_tiles<256, 128, 4, 2, O, WIDE><<<over(p.M, 256) * over(p.N, 128), 512, 0, s>>>(p);
    else product_tiles<256, 256, 2, 4, O, WIDE><<<over(p.M, 256) * over(p.N, 256), 512, 0, s>>>(p);
  } else {
    product_tiles<128, 128, 2, 2, O, WIDE><<<over(p.M, 128) * over(p.N, 128), 256, 0, s>>>(p);
  }
}

}  // namespace

hipError_t launch_product8(const Product8& p, int out_dtype, hipStream_t s) {
  if (out_dtype == 0) launch<float, true>(p, s);
  else launch<Bf16, false>(p, s);
  return hipGetLastError();
}

}  // namespace cssm
