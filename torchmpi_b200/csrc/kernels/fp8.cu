// Matrices in 8 bits with a scale for each block of 128 (fp8.cuh): made along rows, along columns or both ways in one pass, and read back; and
// the product of a few tokens with weights that are kept so.
//
// The operands of a linear layer's three products are x and w along their rows (forward), dz along its rows and w along its columns
// (input gradient), dz and x along their columns (weight gradient): what a gradient or an input is needed for in both directions is
// read once.  A block takes a tile of 128 x 128, a thread 8 x 8 of it: the largest magnitudes of its rows are found by shuffles, those
// of the columns by one exchange through shared memory, and the transposed bytes pass through shared memory so that they leave in rows of 128.
#include "fp8.cuh"
#include "gelu.cuh"
#include "pdl.cuh"
#include "sm100_ptx.cuh"
#include "vec.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>
#include <type_traits>

namespace tmpi {
namespace fp8 {

using act8::inverse;
using act8::pack2;
using act8::scale_byte;
using act8::value;

// Eight elements as words: magnitudes of 16-bit types are compared two at a time.  `largest` gives the larger magnitude, with a sign that means nothing, and NaN if
// either is.
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
  static constexpr int WORDS = 4;
  static constexpr uint32_t ABS = 0x7fff7fffu, INF = 0x7f80u;
  static __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float get(const uint32_t* w, int k) { return __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return attn_util::pack_bf16(__float_as_uint(lo), __float_as_uint(hi)); }
};
template <> struct Eight<__half> {
  static constexpr int WORDS = 4;
  static constexpr uint32_t ABS = 0x7fff7fffu, INF = 0x7c00u;
  static __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float get(const uint32_t* w, int k) { return __half2float(__ushort_as_half((unsigned short)(w[k >> 1] >> (16 * (k & 1))))); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Eight<float> {
  static constexpr int WORDS = 8;
  static constexpr uint32_t ABS = 0x7fffffffu, INF = 0x7f800000u;
  static __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) {
    float r;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(r);
  }
  static __device__ __forceinline__ float get(const uint32_t* w, int k) { return __uint_as_float(w[k]); }
};
// the largest magnitude in a word, as the type's bits, and the bits of the fp32 number that it is
template <typename T> __device__ __forceinline__ uint32_t of_word(uint32_t w) {
  w &= Eight<T>::ABS;
  return sizeof(T) == 2 ? max(w & 0xffffu, w >> 16) : w;
}
template <typename T> __device__ __forceinline__ uint32_t as_fp32(uint32_t bits);
template <> __device__ __forceinline__ uint32_t as_fp32<__nv_bfloat16>(uint32_t b) { return b << 16; }
template <> __device__ __forceinline__ uint32_t as_fp32<__half>(uint32_t b) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)b))); }
template <> __device__ __forceinline__ uint32_t as_fp32<float>(uint32_t b) { return b; }
// the same word with zeros for what is not finite
template <typename T> __device__ __forceinline__ uint32_t finite_part(uint32_t w) {
  const uint32_t m = w & Eight<T>::ABS;
  if (sizeof(T) == 2) return ((m & 0xffffu) < Eight<T>::INF ? m & 0xffffu : 0u) | ((m >> 16) < Eight<T>::INF ? m & 0xffff0000u : 0u);
  return m < Eight<T>::INF ? m : 0u;
}

// Up to N elements from anywhere, in two steps, so that the loads of several are under way together: the pieces of 16 bytes that hold them (each holds at least one,
// so that it lies in memory that is there; without any, that of `some` element), then shifted by words and by a half, with zeros behind the n-th.
template <typename T, int N> struct Raw {
  static constexpr int WORDS = N * sizeof(T) / 4, PIECES = WORDS / 4 + 1;
  uint4 u[PIECES];
  uint32_t off;
};
template <int N, typename T>
__device__ __forceinline__ Raw<T, N> issue(const T* __restrict__ p, int n, const T* __restrict__ some) {
  Raw<T, N> r;
  const uintptr_t at = (uintptr_t)(n > 0 ? p : some);
  r.off = (uint32_t)at & 15;
  const int last = n > 0 ? (int)(r.off + n * sizeof(T) - 1) >> 4 : 0;
  const uint4* from = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
#pragma unroll
  for (int j = 0; j < Raw<T, N>::PIECES; ++j) r.u[j] = from[min(j, last)];
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void settle(const Raw<T, N>& r, int n, uint32_t (&w)[Raw<T, N>::WORDS]) {
  constexpr int W = Raw<T, N>::WORDS;
  uint32_t c[W + 4];
#pragma unroll
  for (int j = 0; j < Raw<T, N>::PIECES; ++j) c[4 * j] = r.u[j].x, c[4 * j + 1] = r.u[j].y, c[4 * j + 2] = r.u[j].z, c[4 * j + 3] = r.u[j].w;
#pragma unroll
  for (int j = 0; j < W + 2; ++j) c[j] = r.off & 8 ? c[j + 2] : c[j];
#pragma unroll
  for (int j = 0; j < W + 1; ++j) c[j] = r.off & 4 ? c[j + 1] : c[j];
#pragma unroll
  for (int j = 0; j < W; ++j) w[j] = sizeof(T) == 2 ? __funnelshift_r(c[j], c[j + 1], (r.off & 2) * 8) : c[j];
  if (n < N) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if (sizeof(T) == 2 && 2 * j + 1 == n) w[j] &= 0xffffu;
      else if (j * 4 >= n * (int)sizeof(T)) w[j] = 0u;
    }
  }
}

// n elements (up to 8) at p, on a 16-byte boundary
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, uint32_t* w) {
  constexpr int W = Eight<T>::WORDS;
  if (n == 8) {
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + j);
      w[j] = u.x, w[j + 1] = u.y, w[j + 2] = u.z, w[j + 3] = u.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) {
        if constexpr (sizeof(T) == 2) w[k >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(p)[k] << (16 * (k & 1));
        else w[k] = reinterpret_cast<const uint32_t*>(p)[k];
      }
  }
}
template <typename T>
__device__ __forceinline__ void load_whole(const T* __restrict__ p, uint32_t* w) {
#pragma unroll
  for (int j = 0; j < Eight<T>::WORDS; j += 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + j);
    w[j] = u.x, w[j + 1] = u.y, w[j + 2] = u.z, w[j + 3] = u.w;
  }
}

// four values in a word; FINITE: none is infinite
template <bool FINITE>
__device__ __forceinline__ uint32_t four(float a, float b, float c, float d, float inv) {
  if (FINITE) {
    const unsigned long long inv2 = attn_util::pack2(__float_as_uint(inv), __float_as_uint(inv));
    float2 v, u;
    attn_util::unpack2(attn_util::mul2(attn_util::pack2(__float_as_uint(a), __float_as_uint(b)), inv2), v.x, v.y);
    attn_util::unpack2(attn_util::mul2(attn_util::pack2(__float_as_uint(c), __float_as_uint(d)), inv2), u.x, u.y);
    return (uint32_t)__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(u, __NV_SATFINITE, __NV_E4M3) << 16;
  }
  return pack2(a, b, inv) | pack2(c, d, inv) << 16;
}
template <typename T, bool FINITE>
__device__ __forceinline__ uint2 eight(const uint32_t* w, float inv) {
  using E = Eight<T>;
  return make_uint2(four<FINITE>(E::get(w, 0), E::get(w, 1), E::get(w, 2), E::get(w, 3), inv), four<FINITE>(E::get(w, 4), E::get(w, 5), E::get(w, 6), E::get(w, 7), inv));
}

// ---------------------------------------------------------------- along rows
// Eight threads to a block of 128, sixteen elements each, two of a thread's pieces under way at a time (16 bytes by each thread, so that a warp's loads
// are whole lines, took more instructions for an element and 25.7 us in place of 18.1 at 8192 x 4096; now 16.7 - 17.0, fp32 29.1; out of a cold L2 24.6 and 34.8, 65536 x 1024 41.0 and 63.5).  Bound by memory and instructions alike (66 % of
// the issue slots, 0.92 of the copy rate).  VEC: rows start on 16-byte boundaries (else 8192 x 4001 takes 21.9, by elements it took 42).
constexpr int ROW_THREADS = 256;
struct Stride { int rows, pieces; };          // a launch's threads, as rows of pieces (or elements): what a thread's next piece lies further

template <typename T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS) quantize_rows_kernel(const T* __restrict__ x, const long long ld, uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                                                                    const long long rows, const int cols, const Stride step) {
  constexpr int AHEAD = sizeof(T) == 2 ? 2 : 1, W = Eight<T>::WORDS;
  using E = Eight<T>;
  wait_previous(x);
  const int groups = groups_of(cols), per_row = blocks_of(cols) * 8;
  const long long pitch = pitch_of(cols), items = rows * per_row, stride = (long long)gridDim.x * ROW_THREADS;
  long long at = ((long long)blockIdx.x * ROW_THREADS + threadIdx.x) / per_row;
  int piece = (int)((long long)blockIdx.x * ROW_THREADS + threadIdx.x - at * per_row);
  for (long long i0 = (long long)blockIdx.x * ROW_THREADS + threadIdx.x; (i0 & ~31LL) < items; i0 += AHEAD * stride) {
    uint32_t w[AHEAD][2 * W];
    Raw<T, 16> raw[AHEAD];
    long long row[AHEAD];
    int col[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      row[u] = at;
      col[u] = piece * 16;
      const int n = at < rows ? cols - col[u] : 0;
      const T* from = x + row[u] * ld + col[u];
      if (VEC) {
        load8<T>(from, min(8, max(0, n)), w[u]);
        load8<T>(from + 8, min(8, max(0, n - 8)), w[u] + W);
      } else {
        raw[u] = issue<16>(from, min(16, n), x);
      }
      at += step.rows;
      piece += step.pieces;
      if (piece >= per_row) { piece -= per_row; ++at; }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (!VEC) settle(raw[u], row[u] < rows ? cols - col[u] : 0, w[u]);
      uint32_t a = 0;
#pragma unroll
      for (int j = 0; j < 2 * W; ++j) a = E::largest(a, w[u][j]);
      a = of_word<T>(a);
      const bool finite = __all_sync(~0u, a < E::INF);
      if (!finite) {
        a = 0;
#pragma unroll
        for (int j = 0; j < 2 * W; ++j) a = max(a, of_word<T>(finite_part<T>(w[u][j])));
      }
      a = max(a, __shfl_xor_sync(~0u, a, 1));
      a = max(a, __shfl_xor_sync(~0u, a, 2));
      a = max(a, __shfl_xor_sync(~0u, a, 4));
      if (row[u] >= rows) continue;
      const uint32_t byte = scale_byte(as_fp32<T>(a));
      const float inv = inverse(byte);
      uint2 lo, hi;
      if (finite) lo = eight<T, true>(w[u], inv), hi = eight<T, true>(w[u] + W, inv);
      else lo = eight<T, false>(w[u], inv), hi = eight<T, false>(w[u] + W, inv);
      *reinterpret_cast<uint4*>(q + row[u] * pitch + col[u]) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      if ((threadIdx.x & 7) == 0) scale[scale_at(row[u], col[u] / BLOCK, groups)] = (uint8_t)byte;
    }
  }
}

// ---------------------------------------------------------------- along columns, or both
constexpr int TILE = 128, TILE_THREADS = 256, TILE_WARPS = TILE_THREADS / 32, ROWS = 8;

// One matrix, or two in one launch (the input and the weight of a layer): the blocks from a's tiles on take b's.
// GELU: x is the gradient behind a GELU of z; what is kept is x gelu'(z), rounded to T.  q, scale: along the rows, or null.  sums: the columns'
// sums over this tile's rows, [row tiles, cols], or null; both are of a alone.  VEC: rows start on 16-byte boundaries.
// 8192 x 4096 bf16: 24.9 us both ways, out of a cold L2 28.6 (0.82 and 0.72 of the copy rate; along columns alone 18.3 and 24.6; fp32 34.9 and 38.9; 57 % of the issue slots, of a warp's time two fifths waiting for its loads), with the sums 26.8, with the GELU's
// gradient and the sums 53 (0.58; 28 million warp instructions, by four warps to a scheduler).  40 us both ways where rows start anywhere (8192 x 4001).
template <typename T> struct Matrix {
  const T* x;
  long long ld;
  uint8_t *q, *scale, *qt, *scalet;
  int rows, cols;
};
template <typename T, bool GELU, bool VEC>
__global__ void __launch_bounds__(TILE_THREADS, sizeof(T) == 4 || GELU || !VEC ? 2 : 3)
quantize_tiles_kernel(const Matrix<T> a, const Matrix<T> b, const T* __restrict__ z, float* __restrict__ sums_of_a) {
  using E = Eight<T>;
  constexpr int W = E::WORDS, R = sizeof(T) == 2 ? 4 : 2;          // rows of a thread whose pieces are under way together
  __shared__ __align__(16) uint32_t tops[TILE_WARPS][16 * W];
  __shared__ __align__(16) float part[TILE_WARPS][TILE];
  __shared__ __align__(16) float column_inv[TILE];
  __shared__ __align__(16) uint8_t turned[TILE * TILE];
  const int tiles_of_a = blocks_of(a.cols) * blocks_of(a.rows);
  const bool second = (int)blockIdx.x >= tiles_of_a;
  const T* x = second ? b.x : a.x;
  wait_previous(x, z);
  const long long ld = second ? b.ld : a.ld;
  uint8_t *const q = second ? b.q : a.q, *const scale = second ? b.scale : a.scale, *const qt = second ? b.qt : a.qt, *const scalet = second ? b.scalet : a.scalet;
  float* const sums = second ? nullptr : sums_of_a;
  const int rows = second ? b.rows : a.rows, cols = second ? b.cols : a.cols;
  const int t = threadIdx.x, cg = t & 15, rg = t >> 4, warp = t >> 5, tile = (int)blockIdx.x - (second ? tiles_of_a : 0);
  const int col_tiles = blocks_of(cols), cb = tile % col_tiles, rb = tile / col_tiles;
  const int row0 = rb * TILE + rg * ROWS, col0 = cb * TILE + cg * 8, n = max(0, min(8, cols - col0));
  const bool whole = (cb + 1) * TILE <= cols && (rb + 1) * TILE <= rows;
  uint32_t w[ROWS][W];
  const T* from = x + (long long)row0 * ld + col0;
  if (VEC && whole) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) load_whole<T>(from + i * ld, w[i]);
  } else if (VEC) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) load8<T>(from + i * ld, row0 + i < rows ? n : 0, w[i]);
  } else {
#pragma unroll
    for (int h = 0; h < ROWS; h += R) {
      Raw<T, 8> raw[R];
#pragma unroll
      for (int i = 0; i < R; ++i) raw[i] = issue<8>(from + (h + i) * ld, row0 + h + i < rows ? n : 0, x);
#pragma unroll
      for (int i = 0; i < R; ++i) settle(raw[i], row0 + h + i < rows ? n : 0, w[h + i]);
    }
  }
  if constexpr (GELU) {
    const T* z0 = z + (long long)row0 * cols + col0;
#pragma unroll
    for (int h = 0; h < ROWS; h += 4) {                   // z four rows at a time
      uint32_t zs[4][W];
      if (VEC && whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load_whole<T>(z0 + (long long)(h + i) * cols, zs[i]);
      } else if (VEC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load8<T>(z0 + (long long)(h + i) * cols, row0 + h + i < rows ? n : 0, zs[i]);
      } else {
#pragma unroll
        for (int g = 0; g < 4; g += R) {
          Raw<T, 8> raw[R];
#pragma unroll
          for (int i = 0; i < R; ++i) raw[i] = issue<8>(z0 + (long long)(h + g + i) * cols, row0 + h + g + i < rows ? n : 0, z);
#pragma unroll
          for (int i = 0; i < R; ++i) settle(raw[i], row0 + h + g + i < rows ? n : 0, zs[g + i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          uint32_t* v = w[h + i];
          unsigned long long slope;
          if constexpr (std::is_same_v<T, __nv_bfloat16>) {          // results of 8 bits: the quicker form (gelu.cuh)
            slope = quick_gelu_slope2(attn_util::pack2(__float_as_uint(E::get(zs[i], k)), __float_as_uint(E::get(zs[i], k + 1))));
          } else {
            float s0, s1;
            gelu_grad2(E::get(zs[i], k), E::get(zs[i], k + 1), &s0, &s1);
            slope = attn_util::pack2(__float_as_uint(s0), __float_as_uint(s1));
          }
          float d0, d1;
          attn_util::unpack2(attn_util::mul2(slope, attn_util::pack2(__float_as_uint(E::get(v, k)), __float_as_uint(E::get(v, k + 1)))), d0, d1);
          if constexpr (sizeof(T) == 2) v[k >> 1] = E::pack(d0, d1);
          else v[k] = __float_as_uint(d0), v[k + 1] = __float_as_uint(d1);
        }
    }
  }
  uint32_t top_row[ROWS], top_col[W];
#pragma unroll
  for (int j = 0; j < W; ++j) top_col[j] = 0;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    top_row[i] = 0;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      top_row[i] = E::largest(top_row[i], w[i][j]);
      top_col[j] = E::largest(top_col[j], w[i][j]);
    }
  }
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) all = max(all, top_row[i] = of_word<T>(top_row[i]));
  const bool finite = __syncthreads_and(all < E::INF);      // of the whole tile: both directions take the same elements
  if (!finite) {                                            // what is not finite has no say about the scales
#pragma unroll
    for (int j = 0; j < W; ++j) top_col[j] = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      top_row[i] = 0;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        top_row[i] = max(top_row[i], of_word<T>(finite_part<T>(w[i][j])));
        top_col[j] = E::largest(top_col[j], finite_part<T>(w[i][j]));
      }
    }
  }
  if (sums) {
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      unsigned long long a = attn_util::pack2(0u, 0u);
#pragma unroll
      for (int i = 0; i < ROWS; ++i) a = attn_util::add2(a, attn_util::pack2(__float_as_uint(E::get(w[i], k)), __float_as_uint(E::get(w[i], k + 1))));
      attn_util::unpack2(a, s[k], s[k + 1]);
      s[k] += __shfl_xor_sync(~0u, s[k], 16);
      s[k + 1] += __shfl_xor_sync(~0u, s[k + 1], 16);
    }
    if (!(t & 16)) {
      *reinterpret_cast<float4*>(&part[warp][cg * 8]) = make_float4(s[0], s[1], s[2], s[3]);
      *reinterpret_cast<float4*>(&part[warp][cg * 8 + 4]) = make_float4(s[4], s[5], s[6], s[7]);
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) top_col[j] = E::largest(top_col[j], __shfl_xor_sync(~0u, top_col[j], 16));
  if (!(t & 16)) {
#pragma unroll
    for (int j = 0; j < W; j += 4) *reinterpret_cast<uint4*>(&tops[warp][cg * W + j]) = make_uint4(top_col[j], top_col[j + 1], top_col[j + 2], top_col[j + 3]);
  }
  if (q) {
    // The 16 threads of a row exchange halves of their rows' maxima: lane cg is left with that of row cg / 2, whose scale it forms, and all take the
    // eight scales from there.
    uint32_t m[4];
    const bool up8 = cg & 8, up4 = cg & 4, up2 = cg & 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max(up8 ? top_row[4 + i] : top_row[i], __shfl_xor_sync(~0u, up8 ? top_row[i] : top_row[4 + i], 8));
#pragma unroll
    for (int i = 0; i < 2; ++i) m[i] = max(up4 ? m[2 + i] : m[i], __shfl_xor_sync(~0u, up4 ? m[i] : m[2 + i], 4));
    m[0] = max(up2 ? m[1] : m[0], __shfl_xor_sync(~0u, up2 ? m[0] : m[1], 2));
    m[0] = max(m[0], __shfl_xor_sync(~0u, m[0], 1));
    const uint32_t byte = scale_byte(as_fp32<T>(m[0]));
    if (!(cg & 1)) scale[scale_at(row0 + (cg >> 1), cb, groups_of(cols))] = (uint8_t)byte;
    const long long pitch = pitch_of(cols);
    uint8_t* to = q + row0 * pitch + col0;
    float inv[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) inv[i] = inverse(__shfl_sync(~0u, byte, (t & 16) + 2 * i));
    if (finite && whole) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) *reinterpret_cast<uint2*>(to + i * pitch) = eight<T, true>(w[i], inv[i]);
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (row0 + i < rows) *reinterpret_cast<uint2*>(to + i * pitch) = finite ? eight<T, true>(w[i], inv[i]) : eight<T, false>(w[i], inv[i]);
    }
  }
  __syncthreads();
  // the columns' maxima over the warps, a word by each of the first threads, and their scales
  if (t < 16 * W) {
    uint32_t m = tops[0][t];
#pragma unroll
    for (int v = 1; v < TILE_WARPS; ++v) m = E::largest(m, tops[v][t]);
    m &= E::ABS;
    const int c = sizeof(T) == 2 ? 2 * t : t;
    uint8_t* to = scalet + scale_at(cb * TILE + c, rb, groups_of(rows));          // a column further: 16 bytes (an even column never ends a group of 32)
    const uint32_t byte = scale_byte(as_fp32<T>(sizeof(T) == 2 ? m & 0xffffu : m));
    to[0] = (uint8_t)byte;
    column_inv[c] = inverse(byte);
    if (sizeof(T) == 2) {
      const uint32_t odd = scale_byte(as_fp32<T>(m >> 16));
      to[16] = (uint8_t)odd;
      column_inv[c + 1] = inverse(odd);
    }
  }
  __syncthreads();
  float inv[8];
  *reinterpret_cast<float4*>(&inv[0]) = *reinterpret_cast<const float4*>(&column_inv[cg * 8]);
  *reinterpret_cast<float4*>(&inv[4]) = *reinterpret_cast<const float4*>(&column_inv[cg * 8 + 4]);
  // eight rows of column col0 + k; pieces of 8 bytes change places by the column's group, so that the 16 threads that store together hit all banks
  uint8_t* to = &turned[cg * 8 * TILE + ((rg ^ cg) << 3)];
  if (finite) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      *reinterpret_cast<uint2*>(to + k * TILE) = make_uint2(four<true>(E::get(w[0], k), E::get(w[1], k), E::get(w[2], k), E::get(w[3], k), inv[k]),
                                                            four<true>(E::get(w[4], k), E::get(w[5], k), E::get(w[6], k), E::get(w[7], k), inv[k]));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      *reinterpret_cast<uint2*>(to + k * TILE) = make_uint2(four<false>(E::get(w[0], k), E::get(w[1], k), E::get(w[2], k), E::get(w[3], k), inv[k]),
                                                            four<false>(E::get(w[4], k), E::get(w[5], k), E::get(w[6], k), E::get(w[7], k), inv[k]));
  }
  __syncthreads();
  const long long pitch_t = pitch_of(rows);
  uint8_t* out = qt + (cb * TILE + (t >> 4)) * pitch_t + rb * TILE + (t & 15) * 8;
  // column (t >> 4) + 16 j: its group is (t >> 7) + 2 j
  const uint8_t* piece = &turned[(t >> 4) * TILE];
  if (whole) {
#pragma unroll
    for (int j = 0; j < TILE / 16; ++j)
      *reinterpret_cast<uint2*>(out + 16 * j * pitch_t) = *reinterpret_cast<const uint2*>(piece + 16 * j * TILE + (((t & 15) ^ ((t >> 7) + 2 * j)) << 3));
  } else {
#pragma unroll
    for (int j = 0; j < TILE / 16; ++j)
      if (cb * TILE + (t >> 4) + 16 * j < cols)
        *reinterpret_cast<uint2*>(out + 16 * j * pitch_t) = *reinterpret_cast<const uint2*>(piece + 16 * j * TILE + (((t & 15) ^ ((t >> 7) + 2 * j)) << 3));
  }
  if (sums && t < TILE && cb * TILE + t < cols) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < TILE_WARPS; ++v) s += part[v][t];
    sums[(size_t)rb * cols + cb * TILE + t] = s;
  }
}

// db[c] = the sum of the tiles' sums, in their order
template <typename T>
__global__ void __launch_bounds__(256) column_sums_kernel(const float* __restrict__ sums, const int tiles, const int cols, T* __restrict__ db) {
  wait_previous(sums);
  __shared__ float part[8][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  float s = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int i = g; i < tiles; i += 8) s += sums[(size_t)i * cols + c];
  part[g][threadIdx.x & 31] = s;
  __syncthreads();
  if (g == 0 && c < cols) {
#pragma unroll
    for (int v = 1; v < 8; ++v) s += part[v][threadIdx.x];
    db[c] = from_acc<T>((typename AccOf<T>::type)s);
  }
}

// ---------------------------------------------------------------- back
// 16 bytes of the result by each thread, rows being so many whole pieces.  vec: they are on 16-byte boundaries; the branch also keeps the four loads together (without it 21 us at
// 8192 x 4096 bf16, with it 17).
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) restore_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, T* __restrict__ x, const long long rows, const int cols,
                                                              const bool vec, const Stride step) {
  constexpr int PER = 16 / sizeof(T), AHEAD = 4;
  wait_previous(q, scale);
  const int groups = groups_of(cols);
  const long long pitch = pitch_of(cols), total = rows * cols, stride = (long long)gridDim.x * ROW_THREADS * PER;
  long long first = ((long long)blockIdx.x * ROW_THREADS + threadIdx.x) * PER, at = first / cols;
  int in_row = (int)(first - at * cols);
  for (; first < total; first += AHEAD * stride) {
    uint2 u[AHEAD];
    uint32_t s[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const bool there = first + a * stride < total;
      const long long row = there ? at : 0;
      const int col = there ? in_row : 0;
      at += step.rows;
      in_row += step.pieces;
      if (in_row >= cols) { in_row -= cols; ++at; }
      const uint8_t* p = q + row * pitch + col;
      u[a] = PER == 8 ? *reinterpret_cast<const uint2*>(p) : make_uint2(*reinterpret_cast<const uint32_t*>(p), 0u);
      s[a] = scale[scale_at(row, col / BLOCK, groups)];
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const long long e = first + a * stride;
      if (e >= total) break;
      float f[8];
      act8::unpack8(u[a], value(s[a]), f);
      if (vec) {
        Pack<T, PER> o;
#pragma unroll
        for (int k = 0; k < PER; ++k) o.v[k] = from_acc<T>((typename AccOf<T>::type)f[k]);
        st_pack<T, PER>(x + e, o);
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k) x[e + k] = from_acc<T>((typename AccOf<T>::type)f[k]);
      }
    }
  }
}

// Rows that are not: their first and last pieces are shared with their neighbours' (stored by elements), and a piece's bytes lie anywhere in theirs: whole words, shifted
// (8192 x 4001 bf16 in 31 us, where pieces of rows that were stored by elements took 96; 4096 columns take 17).
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) restore_any_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, T* __restrict__ x, const long long rows, const int cols,
                                                                  const Stride step) {
  constexpr int PER = 16 / sizeof(T), AHEAD = 4;
  wait_previous(q, scale);
  const int groups = groups_of(cols), per_row = (cols + PER - 1) / PER + 1;
  const long long pitch = pitch_of(cols), items = rows * per_row, stride = (long long)gridDim.x * ROW_THREADS;
  long long i0 = (long long)blockIdx.x * ROW_THREADS + threadIdx.x, at = i0 / per_row;
  int piece = (int)(i0 - at * per_row);
  for (; i0 < items; i0 += AHEAD * stride) {
    uint2 u[AHEAD];
    uint32_t s[AHEAD], s_next[AHEAD];
    long long row[AHEAD];
    int col[AHEAD];                    // of the piece's first element: in front of the row's where that is inside a piece
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const bool there = i0 + a * stride < items;
      row[a] = there ? at : 0;
      col[a] = (there ? piece * PER : 0) - (int)((uintptr_t)(x + row[a] * cols) & 15) / (int)sizeof(T);
      at += step.rows;
      piece += step.pieces;
      if (piece >= per_row) { piece -= per_row; ++at; }
      const int from = col[a] & ~3, by = (col[a] & 3) * 8;
      uint32_t w[3];
#pragma unroll
      for (int j = 0; j < 3; ++j)
        w[j] = from + 4 * j >= 0 && from + 4 * j < pitch && (j < 2 || PER == 8) ? *reinterpret_cast<const uint32_t*>(q + row[a] * pitch + from + 4 * j) : 0u;
      u[a] = make_uint2(__funnelshift_r(w[0], w[1], by), __funnelshift_r(w[1], w[2], by));
      s[a] = scale[scale_at(row[a], min(max(col[a], 0), cols - 1) / BLOCK, groups)];
      s_next[a] = scale[scale_at(row[a], min(max(col[a] + PER - 1, 0), cols - 1) / BLOCK, groups)];
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i0 + a * stride >= items) break;
      float f[8];
      act8::unpack8(u[a], 1.f, f);
      const float here = value(s[a]), next = value(s_next[a]);
      const int last = (max(col[a], 0) | (BLOCK - 1)) - col[a];          // of the first block
#pragma unroll
      for (int k = 0; k < PER; ++k) f[k] *= k <= last ? here : next;
      T* p = x + row[a] * cols + col[a];
      if (col[a] >= 0 && col[a] + PER <= cols) {
        Pack<T, PER> o;
#pragma unroll
        for (int k = 0; k < PER; ++k) o.v[k] = from_acc<T>((typename AccOf<T>::type)f[k]);
        st_pack<T, PER>(p, o);
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (col[a] + k >= 0 && col[a] + k < cols) p[k] = from_acc<T>((typename AccOf<T>::type)f[k]);
      }
    }
  }
}

// ---------------------------------------------------------------- a few tokens
// y = x w^T (+ bias, GELU) for up to 32 rows of x and weights in 8 bits, in one launch: bound by reading the weights and by latency.  A block takes
// 16 weight rows, its warps (up to 16) the blocks of K in turn, so that no warp waits for another before the last sum.  A warp
// quantizes the tokens' blocks itself, straight into the operand registers of mma.sync (16 weight rows x 8 tokens x 32 of K): which K
// index stands where is free as long as both operands agree, so a thread's 32 bytes of a weight row are the 32 consecutive ones of its quarter of the
// block, and so are the tokens'.  The sums of a block are scaled into fp32 sums.  The next block's weights are under way meanwhile.
// Few weight rows leave SMs idle: then two or four blocks, a cluster, share the blocks of K, and the first adds what the others leave in its shared memory, in order
// (13 tokens, 4096 -> 1024: 6.5 us, 8.1 without the sharing; 5.7 since a row's pieces are sent for together).  1024 -> 4096: 3.4 us for one token, 7.0 for 32.
constexpr int FEW_ROWS = 16, FEW_WARPS = 16;

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// v 2^(a - 127 + b - 127) without an intermediate result out of range
__device__ __forceinline__ float scaled(float v, uint32_t a, uint32_t b) {
  const uint32_t h = (a + b) >> 1;
  return v * value(h) * value(a + b - h);
}

template <typename T, int NT>
__global__ void __launch_bounds__(FEW_WARPS * 32) few_kernel(const T* __restrict__ x, const long long ld, const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                             const T* __restrict__ bias, T* __restrict__ y, const int tokens, const int N, const int K, const int gelu, const bool vec) {
  using E = Eight<T>;
  constexpr int AT_ONCE = NT == 4 ? (sizeof(T) == 2 ? 2 : 1) : NT;          // groups of eight tokens whose loads are under way together: all of four spilled registers
  __shared__ float part[FEW_WARPS][FEW_ROWS][NT * 8 + 1];
  __shared__ float others[3][FEW_ROWS * NT * 8];
  wait_previous(x, q, scale, bias);
  const int share = blockIdx.y, shares = gridDim.y;          // of the blocks of K; the rank in the cluster
  if (shares > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // started: waited for before its shared memory is written to
  const int lane = threadIdx.x & 31, in_block = threadIdx.x >> 5, warp = in_block * shares + share, warps = (blockDim.x >> 5) * shares, g = lane >> 2, t = lane & 3;
  const int blocks = blocks_of(K), groups = groups_of(K), n0 = blockIdx.x * FEW_ROWS;
  const long long pitch = pitch_of(K);
  const int r0 = min(n0 + g, N - 1), r1 = min(n0 + g + 8, N - 1);
  const uint8_t *w0 = q + r0 * pitch + t * 32, *w1 = q + r1 * pitch + t * 32;
  uint4 next[4];
  uint32_t next_scale[2];
  auto fetch = [&](int b) {
    next[0] = __ldg(reinterpret_cast<const uint4*>(w0 + b * BLOCK));
    next[1] = __ldg(reinterpret_cast<const uint4*>(w0 + b * BLOCK + 16));
    next[2] = __ldg(reinterpret_cast<const uint4*>(w1 + b * BLOCK));
    next[3] = __ldg(reinterpret_cast<const uint4*>(w1 + b * BLOCK + 16));
    next_scale[0] = scale[scale_at(r0, b, groups)];
    next_scale[1] = scale[scale_at(r1, b, groups)];
  };
  if (warp < blocks) fetch(warp);
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = 0.f;
#pragma unroll 1
  for (int b = warp; b < blocks; b += warps) {
    const int col = b * BLOCK + t * 32;
    const uint4 a[4] = {next[0], next[1], next[2], next[3]};
    const uint32_t sw[2] = {next_scale[0], next_scale[1]};
    if (b + warps < blocks) fetch(b + warps);
    uint32_t v[AT_ONCE][4 * E::WORDS];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (i * 8 >= tokens) break;
      if (i % AT_ONCE == 0) {
        const bool whole = vec && col + 32 <= K;
        if (whole) {
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int j = 0; j < 4 * E::WORDS; j += E::WORDS) {
              const int token = min((i + u) * 8 + g, tokens - 1);
              load_whole<T>(x + (long long)token * ld + col + j / E::WORDS * 8, v[u] + j);
            }
        } else {
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u) {
            const int token = min((i + u) * 8 + g, tokens - 1), n = min(32, K - col);
            settle(issue<32>(x + (long long)token * ld + col, n, x), n, v[u]);
          }
        }
      }
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 4 * E::WORDS; ++k) top = E::largest(top, v[i % AT_ONCE][k]);
      top = of_word<T>(top);
      const bool finite = __all_sync(~0u, top < E::INF);
      if (!finite) {
        top = 0;
#pragma unroll
        for (int k = 0; k < 4 * E::WORDS; ++k) top = max(top, of_word<T>(finite_part<T>(v[i % AT_ONCE][k])));
      }
      top = max(top, __shfl_xor_sync(~0u, top, 1));
      top = max(top, __shfl_xor_sync(~0u, top, 2));
      const uint32_t sx = scale_byte(as_fp32<T>(top));
      const float inv = inverse(sx);
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {                    // 8 of the thread's 32 bytes for each of the four instructions
        const uint2 xq = finite ? eight<T, true>(v[i % AT_ONCE] + j * E::WORDS, inv) : eight<T, false>(v[i % AT_ONCE] + j * E::WORDS, inv);
        const uint4 p = a[j >> 1], r = a[2 + (j >> 1)];
        if (j & 1) mma_e4m3(c, p.z, r.z, p.w, r.w, xq.x, xq.y);
        else mma_e4m3(c, p.x, r.x, p.y, r.y, xq.x, xq.y);
      }
      const uint32_t s0 = __shfl_sync(~0u, sx, 8 * t), s1 = __shfl_sync(~0u, sx, 8 * t + 4);      // of the tokens 2 t and 2 t + 1
      acc[i][0] += scaled(c[0], sw[0], s0);
      acc[i][1] += scaled(c[1], sw[0], s1);
      acc[i][2] += scaled(c[2], sw[1], s0);
      acc[i][3] += scaled(c[3], sw[1], s1);
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    part[in_block][g][i * 8 + 2 * t] = acc[i][0];
    part[in_block][g][i * 8 + 2 * t + 1] = acc[i][1];
    part[in_block][g + 8][i * 8 + 2 * t] = acc[i][2];
    part[in_block][g + 8][i * 8 + 2 * t + 1] = acc[i][3];
  }
  __syncthreads();
  if (shares > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (share)
      for (int i = threadIdx.x; i < FEW_ROWS * tokens; i += blockDim.x) {
        float s = 0.f;
        for (int v = 0; v < (int)(blockDim.x >> 5); ++v) s += part[v][i & (FEW_ROWS - 1)][i / FEW_ROWS];
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(sm100::map_to_cta(&others[share - 1][i], 0)), "f"(s) : "memory");
      }
    sm100::cluster_sync();
    if (share) return;
  }
  for (int i = threadIdx.x; i < FEW_ROWS * tokens; i += blockDim.x) {
    const int r = i & (FEW_ROWS - 1), token = i / FEW_ROWS;
    if (n0 + r >= N) continue;
    float s = 0.f;
    for (int v = 0; v < (int)(blockDim.x >> 5); ++v) s += part[v][r][token];
    for (int v = 1; v < shares; ++v) s += others[v - 1][i];
    if (bias) s += (float)to_acc<T>(bias[n0 + r]);
    T out = from_acc<T>((typename AccOf<T>::type)s);
    if (gelu) {
      float y0, y1;
      gelu_value2((float)to_acc<T>(out), 0.f, &y0, &y1);
      out = from_acc<T>((typename AccOf<T>::type)y0);
    }
    y[(long long)token * N + n0 + r] = out;
  }
}

template <typename F>
static int by_type(int dtype, const char* what, F f) {
  cudaError_t e;
  switch (dtype) {
    case TMPI_BF16: e = f((__nv_bfloat16*)nullptr); break;
    case TMPI_F16: e = f((__half*)nullptr); break;
    case TMPI_F32: e = f((float*)nullptr); break;
    default: return fail(TMPI_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  }
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}
static bool whole_pieces(std::initializer_list<const void*> p, int64_t ld, int es) { return all_aligned16(p) && ld * es % 16 == 0; }
// A launch for rows of `per_row` pieces, `ahead` of them by each thread at a time, in at most `most` blocks.
struct RowLaunch { int blocks; Stride step; };
static RowLaunch row_launch(int64_t rows, int per_row, int ahead, int most) {
  const int blocks = (int)std::min<int64_t>((rows * per_row + ahead * ROW_THREADS - 1) / (ahead * ROW_THREADS), most);
  return {blocks, {(int)((int64_t)blocks * ROW_THREADS / per_row), (int)((int64_t)blocks * ROW_THREADS % per_row)}};
}
static int checked(int64_t rows, int64_t cols, const char* what) {
  if (rows < 0 || cols < 1 || rows > (int64_t)1 << 30 || cols > (int64_t)1 << 30) return fail(TMPI_ERR_INVALID, "%s: %lld rows of %lld", what, (long long)rows, (long long)cols);
  return TMPI_OK;
}

}  // namespace fp8
}  // namespace tmpi

using namespace tmpi;

extern "C" {

int64_t tmpi_fp8_pitch(int64_t cols) { return fp8::pitch_of(cols); }
size_t tmpi_fp8_scale_bytes(int64_t rows, int64_t cols) {
  return (size_t)((rows + fp8::TILE_ROWS - 1) / fp8::TILE_ROWS) * fp8::groups_of(cols) * fp8::TILE_BYTES;
}

// x [rows, cols] of `dtype`, rows `ld` elements apart.  q [rows, pitch(cols)] with its scales: along the rows; qt [cols, pitch(rows)]: along the columns, transposed;
// either may be null.  With z (dense), what is quantized is x gelu'(z) rounded to the type, and with sums [ceil(rows / 128), cols] the columns'
// sums of that over 128 rows each are left there: both need qt.
int tmpi_fp8_quantize(const void* x, int64_t ld, const void* z, void* q, void* scale, void* qt, void* scalet, float* sums, int64_t rows, int64_t cols, int dtype, void* stream) {
  int st = fp8::checked(rows, cols, "fp8_quantize");
  if (st || !rows) return st;
  if ((!q && !qt) || (!qt && (z || sums)) || ld < cols) return fail(TMPI_ERR_INVALID, "fp8_quantize: nothing to write, or row pitch %lld for %lld columns", (long long)ld, (long long)cols);
  if (!all_aligned16({q, scale, qt, scalet, sums})) return fail(TMPI_ERR_INVALID, "fp8_quantize: results must be 16-byte aligned");
  cudaStream_t s = (cudaStream_t)stream;
  return fp8::by_type(dtype, "fp8_quantize", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    const bool vec = fp8::whole_pieces({x, z}, ld, sizeof(T)) && (!z || cols * sizeof(T) % 16 == 0);
    if (!qt) {
      const fp8::RowLaunch l = fp8::row_launch(rows, fp8::blocks_of(cols) * 8, sizeof(T) == 2 ? 2 : 1, 148 * 8);
      return launch_overlapped(vec ? fp8::quantize_rows_kernel<T, true> : fp8::quantize_rows_kernel<T, false>, l.blocks, fp8::ROW_THREADS, 0, s, (const T*)x, (long long)ld, (uint8_t*)q,
                               (uint8_t*)scale, (long long)rows, (int)cols, l.step);
    }
    const long long tiles = (long long)fp8::blocks_of(rows) * fp8::blocks_of(cols);
    if (tiles > 0x7fffffffLL) return cudaErrorInvalidValue;
    const fp8::Matrix<T> a{(const T*)x, ld, (uint8_t*)q, (uint8_t*)scale, (uint8_t*)qt, (uint8_t*)scalet, (int)rows, (int)cols};
    const auto kernel = z ? (vec ? fp8::quantize_tiles_kernel<T, true, true> : fp8::quantize_tiles_kernel<T, true, false>)
                          : (vec ? fp8::quantize_tiles_kernel<T, false, true> : fp8::quantize_tiles_kernel<T, false, false>);
    return launch_overlapped(kernel, (unsigned)tiles, fp8::TILE_THREADS, 0, s, a, a, (const T*)z, sums);
  });
}

// Two matrices both ways in one launch.
int tmpi_fp8_quantize_two(const tmpi_fp8_matrix_t* two, int dtype, void* stream) {
  long long tiles = 0;
  for (int i = 0; i < 2; ++i) {
    const tmpi_fp8_matrix_t& m = two[i];
    const int st = fp8::checked(m.rows, m.cols, "fp8_quantize_two");
    if (st) return st;
    if (!m.q || !m.qt || m.ld < m.cols || !m.rows) return fail(TMPI_ERR_INVALID, "fp8_quantize_two: nothing to write, or row pitch %lld for %lld columns", (long long)m.ld, (long long)m.cols);
    if (!all_aligned16({m.q, m.scale, m.qt, m.scalet})) return fail(TMPI_ERR_INVALID, "fp8_quantize_two: results must be 16-byte aligned");
    tiles += (long long)fp8::blocks_of(m.rows) * fp8::blocks_of(m.cols);
  }
  if (tiles > 0x7fffffffLL) return fail(TMPI_ERR_UNSUPPORTED, "fp8_quantize_two: %lld tiles", tiles);
  return fp8::by_type(dtype, "fp8_quantize_two", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    fp8::Matrix<T> m[2];
    bool vec = true;
    for (int i = 0; i < 2; ++i) {
      m[i] = {(const T*)two[i].x, two[i].ld, (uint8_t*)two[i].q, (uint8_t*)two[i].scale, (uint8_t*)two[i].qt, (uint8_t*)two[i].scalet, (int)two[i].rows, (int)two[i].cols};
      vec = vec && fp8::whole_pieces({two[i].x}, two[i].ld, sizeof(T));
    }
    return launch_overlapped(vec ? fp8::quantize_tiles_kernel<T, false, true> : fp8::quantize_tiles_kernel<T, false, false>, (unsigned)tiles, fp8::TILE_THREADS, 0, (cudaStream_t)stream, m[0], m[1], (const T*)nullptr, (float*)nullptr);
  });
}

// db [cols] = the sums of `tiles` rows of sums
int tmpi_fp8_column_sums(const float* sums, int tiles, int cols, void* db, int dtype, void* stream) {
  if (tiles < 0 || cols < 1) return fail(TMPI_ERR_INVALID, "fp8_column_sums: %d rows of %d", tiles, cols);
  return fp8::by_type(dtype, "fp8_column_sums", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    return launch_overlapped(fp8::column_sums_kernel<T>, (cols + 31) / 32, 256, 0, (cudaStream_t)stream, sums, tiles, cols, (T*)db);
  });
}

int tmpi_fp8_restore(const void* q, const void* scale, void* x, int64_t rows, int64_t cols, int dtype, void* stream) {
  int st = fp8::checked(rows, cols, "fp8_restore");
  if (st || !rows) return st;
  if (!all_aligned16({q})) return fail(TMPI_ERR_INVALID, "fp8_restore: the 8-bit numbers must be 16-byte aligned");
  return fp8::by_type(dtype, "fp8_restore", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    constexpr int PER = 16 / sizeof(T);
    if (cols % PER == 0) {
      const int blocks = (int)std::min<int64_t>((rows * cols / PER + 4 * fp8::ROW_THREADS - 1) / (4 * fp8::ROW_THREADS), 1 << 19);
      const int64_t apart = (int64_t)blocks * fp8::ROW_THREADS * PER;          // elements between a thread's pieces
      return launch_overlapped(fp8::restore_kernel<T>, blocks, fp8::ROW_THREADS, 0, (cudaStream_t)stream, (const uint8_t*)q, (const uint8_t*)scale, (T*)x, (long long)rows, (int)cols,
                               all_aligned16({x}), fp8::Stride{(int)(apart / cols), (int)(apart % cols)});
    }
    const fp8::RowLaunch l = fp8::row_launch(rows, (int)((cols + PER - 1) / PER) + 1, 4, 1 << 20);
    return launch_overlapped(fp8::restore_any_kernel<T>, l.blocks, fp8::ROW_THREADS, 0, (cudaStream_t)stream, (const uint8_t*)q, (const uint8_t*)scale, (T*)x, (long long)rows, (int)cols,
                             l.step);
  });
}

int tmpi_fp8_few_tokens(void) { return 32; }
// y [tokens, N] = x w^T (+ bias) (GELU of what is rounded), x [tokens, K] in rows `ld` apart, up to tmpi_fp8_few_tokens() of them; w [N, K] in 8 bits
int tmpi_fp8_few(const void* x, int64_t ld, const void* q, const void* scale, const void* bias, void* y, int tokens, int N, int K, int gelu, int dtype, void* stream) {
  if (tokens < 1 || tokens > tmpi_fp8_few_tokens() || N < 1 || K < 1 || ld < K) return fail(TMPI_ERR_INVALID, "fp8_few: %d tokens, %d x %d", tokens, N, K);
  if (!all_aligned16({q})) return fail(TMPI_ERR_INVALID, "fp8_few: the weights must be 16-byte aligned");
  return fp8::by_type(dtype, "fp8_few", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    const auto kernel = tokens <= 8 ? fp8::few_kernel<T, 1> : tokens <= 16 ? fp8::few_kernel<T, 2> : fp8::few_kernel<T, 4>;
    // Shares of K as long as the blocks fit the SMs and each has blocks of K for half its warps.  More blocks than SMs have eight warps, so that two fit an SM (4 tokens, 4096 -> 4096:
    // 12.3 -> 10.9 us when it was introduced, 7.3 now).
    const int groups = (N + fp8::FEW_ROWS - 1) / fp8::FEW_ROWS, blocks = fp8::blocks_of(K);
    int shares = 1;
    while (shares < 4 && groups * shares * 2 <= 148 && blocks >= shares * fp8::FEW_WARPS) shares *= 2;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 1; at[1].val.clusterDim.y = (unsigned)shares; at[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)groups, (unsigned)shares);
    cfg.blockDim = dim3(32 * std::min(groups > 148 ? fp8::FEW_WARPS / 2 : fp8::FEW_WARPS, (blocks + shares - 1) / shares));
    cfg.stream = (cudaStream_t)stream; cfg.attrs = at; cfg.numAttrs = shares > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, (const T*)x, (long long)ld, (const uint8_t*)q, (const uint8_t*)scale, (const T*)bias, (T*)y, tokens, N, K, gelu,
                              fp8::whole_pieces({x}, ld, sizeof(T)));
  });
}

}  // extern "C"
