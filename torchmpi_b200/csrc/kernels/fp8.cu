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
#include "vec.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>

namespace tmpi {
namespace fp8 {

using act8::inverse;
using act8::magnitude;
using act8::pack2;
using act8::scale_byte;
using act8::value;

// Eight elements as words: magnitudes of 16-bit types are compared two at a time, as integers (which order like the values).
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
  static constexpr int WORDS = 4;
  static constexpr uint32_t ABS = 0x7fff7fffu, INF = 0x7f80u;
  static __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  static __device__ __forceinline__ float get(const uint32_t* w, int k) { return __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return attn_util::pack_bf16(__float_as_uint(lo), __float_as_uint(hi)); }
};
template <> struct Eight<__half> {
  static constexpr int WORDS = 4;
  static constexpr uint32_t ABS = 0x7fff7fffu, INF = 0x7c00u;
  static __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  static __device__ __forceinline__ float get(const uint32_t* w, int k) { return __half2float(__ushort_as_half((unsigned short)(w[k >> 1] >> (16 * (k & 1))))); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Eight<float> {
  static constexpr int WORDS = 8;
  static constexpr uint32_t ABS = 0x7fffffffu, INF = 0x7f800000u;
  static __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ float get(const uint32_t* w, int k) { return __uint_as_float(w[k]); }
};
// the largest magnitude in a word, as the type's bits, and the bits of the fp32 number that it is
template <typename T> __device__ __forceinline__ uint32_t of_word(uint32_t w) { return sizeof(T) == 2 ? max(w & 0xffffu, w >> 16) : w; }
template <typename T> __device__ __forceinline__ uint32_t as_fp32(uint32_t bits);
template <> __device__ __forceinline__ uint32_t as_fp32<__nv_bfloat16>(uint32_t b) { return b << 16; }
template <> __device__ __forceinline__ uint32_t as_fp32<__half>(uint32_t b) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)b))); }
template <> __device__ __forceinline__ uint32_t as_fp32<float>(uint32_t b) { return b; }

// n elements (up to 8) at p; vec: whole, and on 16-byte boundaries
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, bool vec, uint32_t (&w)[Eight<T>::WORDS]) {
  constexpr int W = Eight<T>::WORDS;
  if (vec && n == 8) {
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

// four values in a word; `finite`: none is infinite
__device__ __forceinline__ uint32_t four(float a, float b, float c, float d, float inv, bool finite) {
  if (finite) {
    const unsigned long long inv2 = attn_util::pack2(__float_as_uint(inv), __float_as_uint(inv));
    float2 v, u;
    attn_util::unpack2(attn_util::mul2(attn_util::pack2(__float_as_uint(a), __float_as_uint(b)), inv2), v.x, v.y);
    attn_util::unpack2(attn_util::mul2(attn_util::pack2(__float_as_uint(c), __float_as_uint(d)), inv2), u.x, u.y);
    return (uint32_t)__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(u, __NV_SATFINITE, __NV_E4M3) << 16;
  }
  return pack2(a, b, inv) | pack2(c, d, inv) << 16;
}

// ---------------------------------------------------------------- along rows
// Eight threads to a block of 128, sixteen elements each.
constexpr int ROW_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) quantize_rows_kernel(const T* __restrict__ x, const long long ld, uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                                                                    const long long rows, const int cols, const bool vec) {
  wait_previous(x);
  const int blocks = blocks_of(cols), groups = groups_of(cols);
  const long long pitch = pitch_of(cols), items = rows * blocks * 8, stride = (long long)gridDim.x * ROW_THREADS;
  using E = Eight<T>;
  for (long long i = (long long)blockIdx.x * ROW_THREADS + threadIdx.x; (i & ~31LL) < items; i += stride) {
    const long long per_row = blocks * 8, row = i < items ? i / per_row : 0;
    const int col = (int)(i - row * per_row) * 16, n = i < items ? cols - col : 0;
    uint32_t w[2][E::WORDS];
    load8<T>(x + row * ld + col, min(8, max(0, n)), vec, w[0]);
    load8<T>(x + row * ld + col + 8, min(8, max(0, n - 8)), vec, w[1]);
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < E::WORDS; ++j) a = E::largest(a, E::largest(w[0][j] & E::ABS, w[1][j] & E::ABS));
    a = of_word<T>(a);
    const bool finite = __all_sync(~0u, a < E::INF);
    a = as_fp32<T>(a);
    if (!finite) {
      a = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) a = max(a, magnitude(E::get(w[k >> 3], k & 7)));
    }
    a = max(a, __shfl_xor_sync(~0u, a, 1));
    a = max(a, __shfl_xor_sync(~0u, a, 2));
    a = max(a, __shfl_xor_sync(~0u, a, 4));
    if (i >= items) continue;
    const uint32_t byte = scale_byte(a);
    const float inv = inverse(byte);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t* v = w[j >> 1];
      const int k = 4 * (j & 1);
      o[j] = four(E::get(v, k), E::get(v, k + 1), E::get(v, k + 2), E::get(v, k + 3), inv, finite);
    }
    *reinterpret_cast<uint4*>(q + row * pitch + col) = make_uint4(o[0], o[1], o[2], o[3]);
    if ((threadIdx.x & 7) == 0) scale[scale_at(row, col / BLOCK, groups)] = (uint8_t)byte;
  }
}

// ---------------------------------------------------------------- along columns, or both
constexpr int TILE = 128, TILE_THREADS = 256;

// GELU: x is the gradient behind a GELU of z; what is kept is x gelu'(z), rounded to T.  q, scale: along the rows, or null.  sums: the columns'
// sums over this tile's rows, [row tiles, cols], or null.
template <typename T, bool GELU>
__global__ void __launch_bounds__(TILE_THREADS, sizeof(T) == 2 ? 3 : 2)
quantize_tiles_kernel(const T* __restrict__ x, const long long ld, const T* __restrict__ z, uint8_t* __restrict__ q, uint8_t* __restrict__ scale, uint8_t* __restrict__ qt,
                      uint8_t* __restrict__ scalet, float* __restrict__ sums, const int rows, const int cols, const bool vec) {
  using E = Eight<T>;
  constexpr int W = E::WORDS;
  __shared__ __align__(16) uint32_t tops[8][16 * W];
  __shared__ __align__(16) float part[8][TILE];
  __shared__ __align__(16) uint8_t turned[TILE * TILE];
  wait_previous(x, z);
  const int t = threadIdx.x, cg = t & 15, rg = t >> 4, warp = t >> 5;
  const int col_tiles = blocks_of(cols), cb = (int)(blockIdx.x % col_tiles), rb = (int)(blockIdx.x / col_tiles);
  const int row0 = rb * TILE + rg * 8, col0 = cb * TILE + cg * 8, n = max(0, min(8, cols - col0));
  uint32_t w[8][W];
#pragma unroll
  for (int i = 0; i < 8; ++i) load8<T>(x + (long long)(row0 + i) * ld + col0, row0 + i < rows ? n : 0, vec, w[i]);
  if constexpr (GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t u[W];
      load8<T>(z + (long long)(row0 + i) * cols + col0, row0 + i < rows ? n : 0, vec, u);
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        float d0, d1;
        gelu_grad2(E::get(u, k), E::get(u, k + 1), &d0, &d1);
        d0 *= E::get(w[i], k);
        d1 *= E::get(w[i], k + 1);
        if constexpr (sizeof(T) == 2) w[i][k >> 1] = E::pack(d0, d1);
        else w[i][k] = __float_as_uint(d0), w[i][k + 1] = __float_as_uint(d1);
      }
    }
  }
  uint32_t top_row[8], top_col[W], all = 0;
#pragma unroll
  for (int j = 0; j < W; ++j) top_col[j] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t m = w[i][j] & E::ABS;
      a = E::largest(a, m);
      top_col[j] = E::largest(top_col[j], m);
    }
    top_row[i] = of_word<T>(a);
    all = max(all, top_row[i]);
  }
  const bool finite = __syncthreads_and(all < E::INF);      // of the whole tile: both directions take the same elements
  if (!finite) {                                            // what is not finite has no say about the scales
#pragma unroll
    for (int j = 0; j < W; ++j) top_col[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top_row[i] = 0;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        uint32_t m = w[i][j] & E::ABS;
        if (sizeof(T) == 2) m = ((m & 0xffffu) < E::INF ? m & 0xffffu : 0u) | ((m >> 16) < E::INF ? m & 0xffff0000u : 0u);
        else m = m < E::INF ? m : 0u;
        top_col[j] = E::largest(top_col[j], m);
        top_row[i] = max(top_row[i], of_word<T>(m));
      }
    }
  }
  if (sums) {
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[k] += E::get(w[i], k);
      s[k] += __shfl_xor_sync(~0u, s[k], 16);
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
    const int groups = groups_of(cols);
    const long long pitch = pitch_of(cols);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t a = top_row[i];
#pragma unroll
      for (int d = 1; d < 16; d *= 2) a = max(a, __shfl_xor_sync(~0u, a, d));
      const uint32_t byte = scale_byte(as_fp32<T>(a));
      const float inv = inverse(byte);
      if (cg == 0) scale[scale_at(row0 + i, cb, groups)] = (uint8_t)byte;
      if (row0 + i < rows)
        *reinterpret_cast<uint2*>(q + (row0 + i) * pitch + col0) =
            make_uint2(four(E::get(w[i], 0), E::get(w[i], 1), E::get(w[i], 2), E::get(w[i], 3), inv, finite),
                       four(E::get(w[i], 4), E::get(w[i], 5), E::get(w[i], 6), E::get(w[i], 7), inv, finite));
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < W; j += 4) {
    uint4 m = *reinterpret_cast<const uint4*>(&tops[0][cg * W + j]);
#pragma unroll
    for (int v = 1; v < 8; ++v) {
      const uint4 u = *reinterpret_cast<const uint4*>(&tops[v][cg * W + j]);
      m.x = E::largest(m.x, u.x), m.y = E::largest(m.y, u.y), m.z = E::largest(m.z, u.z), m.w = E::largest(m.w, u.w);
    }
    top_col[j] = m.x, top_col[j + 1] = m.y, top_col[j + 2] = m.z, top_col[j + 3] = m.w;
  }
  const int groups_t = groups_of(rows);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t a = sizeof(T) == 2 ? (top_col[k >> 1] >> (16 * (k & 1))) & 0xffffu : top_col[k & (W - 1)];
    const uint32_t byte = scale_byte(as_fp32<T>(a));
    const float inv = inverse(byte);
    if (rg == 0) scalet[scale_at(col0 + k, rb, groups_t)] = (uint8_t)byte;
    // eight rows of column col0 + k; pieces of 8 bytes change places by the column's group, so that the 16 threads that store together hit all banks
    *reinterpret_cast<uint2*>(&turned[(cg * 8 + k) * TILE + ((rg ^ cg) << 3)]) =
        make_uint2(four(E::get(w[0], k), E::get(w[1], k), E::get(w[2], k), E::get(w[3], k), inv, finite),
                   four(E::get(w[4], k), E::get(w[5], k), E::get(w[6], k), E::get(w[7], k), inv, finite));
  }
  __syncthreads();
  const long long pitch_t = pitch_of(rows);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = (t >> 4) + 16 * j, ch = t & 15;
    if (cb * TILE + c < cols)
      *reinterpret_cast<uint2*>(qt + (cb * TILE + c) * pitch_t + rb * TILE + ch * 8) = *reinterpret_cast<const uint2*>(&turned[c * TILE + ((ch ^ (c >> 3)) << 3)]);
  }
  if (sums && t < TILE && cb * TILE + t < cols) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < 8; ++v) s += part[v][t];
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
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) restore_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, T* __restrict__ x, const long long rows, const int cols,
                                                              const bool vec) {
  wait_previous(q, scale);
  const int blocks = blocks_of(cols), groups = groups_of(cols);
  const long long pitch = pitch_of(cols), items = rows * blocks * 8, stride = (long long)gridDim.x * ROW_THREADS;
  for (long long i = (long long)blockIdx.x * ROW_THREADS + threadIdx.x; i < items; i += stride) {
    const long long row = i / (blocks * 8);
    const int col = (int)(i - row * (blocks * 8)) * 16, n = cols - col;
    if (n <= 0) continue;
    const uint4 u = *reinterpret_cast<const uint4*>(q + row * pitch + col);
    const float s = value(scale[scale_at(row, col / BLOCK, groups)]);
    float f[2][8];
    act8::unpack8(make_uint2(u.x, u.y), s, f[0]);
    act8::unpack8(make_uint2(u.z, u.w), s, f[1]);
    T* p = x + row * cols + col;
    if (vec && n >= 16) {
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 16 / V; ++j) {
        Pack<T, V> a;
#pragma unroll
        for (int k = 0; k < V; ++k) a.v[k] = from_acc<T>((typename AccOf<T>::type)f[(j * V + k) >> 3][(j * V + k) & 7]);
        st_pack<T, V>(p + j * V, a);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k < n) p[k] = from_acc<T>((typename AccOf<T>::type)f[k >> 3][k & 7]);
    }
  }
}

// ---------------------------------------------------------------- a few tokens
// y = x w^T (+ bias, GELU) for up to 32 rows of x and weights in 8 bits, in one launch: bound by reading the weights and by latency.  A block takes
// 16 weight rows, its eight warps the blocks of K in turn, so that no warp waits for another before the last sum.  A warp
// quantizes the tokens' blocks itself, straight into the operand registers of mma.sync (16 weight rows x 8 tokens x 32 of K): which K
// index stands where is free as long as both operands agree, so a thread's 32 bytes of a weight row are the 32 consecutive ones of its quarter of the
// block, and so are the tokens'.  The sums of a block are scaled into fp32 sums.
constexpr int FEW_ROWS = 16, FEW_WARPS = 8, FEW_AHEAD = 4;

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
  __shared__ float part[FEW_WARPS][FEW_ROWS][NT * 8 + 1];
  wait_previous(x, q, scale, bias);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int blocks = blocks_of(K), groups = groups_of(K), n0 = blockIdx.x * FEW_ROWS;
  const long long pitch = pitch_of(K);
  const int r0 = min(n0 + g, N - 1), r1 = min(n0 + g + 8, N - 1);
  const uint8_t *w0 = q + r0 * pitch + t * 32, *w1 = q + r1 * pitch + t * 32;
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = 0.f;
  for (int b0 = warp; b0 < blocks; b0 += FEW_WARPS * FEW_AHEAD) {
    uint4 a[FEW_AHEAD][4];
    uint32_t sw[FEW_AHEAD][2];
#pragma unroll
    for (int u = 0; u < FEW_AHEAD; ++u) {
      const int b = b0 + u * FEW_WARPS;
      if (b < blocks) {
        a[u][0] = __ldg(reinterpret_cast<const uint4*>(w0 + b * BLOCK));
        a[u][1] = __ldg(reinterpret_cast<const uint4*>(w0 + b * BLOCK + 16));
        a[u][2] = __ldg(reinterpret_cast<const uint4*>(w1 + b * BLOCK));
        a[u][3] = __ldg(reinterpret_cast<const uint4*>(w1 + b * BLOCK + 16));
        sw[u][0] = scale[scale_at(r0, b, groups)];
        sw[u][1] = scale[scale_at(r1, b, groups)];
      }
    }
#pragma unroll
    for (int u = 0; u < FEW_AHEAD; ++u) {
      const int b = b0 + u * FEW_WARPS;
      if (b >= blocks) break;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (i * 8 >= tokens) break;
        const int token = i * 8 + g, col = b * BLOCK + t * 32;
        uint32_t v[4][E::WORDS], top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          load8<T>(x + (long long)token * ld + col + 8 * j, token < tokens ? min(8, max(0, K - col - 8 * j)) : 0, vec, v[j]);
#pragma unroll
          for (int k = 0; k < E::WORDS; ++k) top = E::largest(top, v[j][k] & E::ABS);
        }
        top = of_word<T>(top);
        const bool finite = __all_sync(~0u, top < E::INF);
        top = as_fp32<T>(top);
        if (!finite) {
          top = 0;
#pragma unroll
          for (int k = 0; k < 32; ++k) top = max(top, magnitude(E::get(v[k >> 3], k & 7)));
        }
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const uint32_t sx = scale_byte(top);
        const float inv = inverse(sx);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {                    // 8 of the thread's 32 bytes for each of the four instructions
          const uint32_t x0 = four(E::get(v[j], 0), E::get(v[j], 1), E::get(v[j], 2), E::get(v[j], 3), inv, finite);
          const uint32_t x1 = four(E::get(v[j], 4), E::get(v[j], 5), E::get(v[j], 6), E::get(v[j], 7), inv, finite);
          const uint4 p = a[u][j >> 1], r = a[u][2 + (j >> 1)];
          if (j & 1) mma_e4m3(c, p.z, r.z, p.w, r.w, x0, x1);
          else mma_e4m3(c, p.x, r.x, p.y, r.y, x0, x1);
        }
        const uint32_t s0 = __shfl_sync(~0u, sx, 8 * t), s1 = __shfl_sync(~0u, sx, 8 * t + 4);      // of the tokens 2 t and 2 t + 1
        acc[i][0] += scaled(c[0], sw[u][0], s0);
        acc[i][1] += scaled(c[1], sw[u][0], s1);
        acc[i][2] += scaled(c[2], sw[u][1], s0);
        acc[i][3] += scaled(c[3], sw[u][1], s1);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    part[warp][g][i * 8 + 2 * t] = acc[i][0];
    part[warp][g][i * 8 + 2 * t + 1] = acc[i][1];
    part[warp][g + 8][i * 8 + 2 * t] = acc[i][2];
    part[warp][g + 8][i * 8 + 2 * t + 1] = acc[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < FEW_ROWS * NT * 8; i += FEW_WARPS * 32) {
    const int r = i & (FEW_ROWS - 1), token = i / FEW_ROWS;
    if (token >= tokens || n0 + r >= N) continue;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < FEW_WARPS; ++v) s += part[v][r][token];
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
static int row_grid(int64_t rows, int cols) {
  return (int)std::min<int64_t>((rows * blocks_of(cols) * 8 + ROW_THREADS - 1) / ROW_THREADS, 148 * 8);
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
    if (!qt)
      return launch_overlapped(fp8::quantize_rows_kernel<T>, fp8::row_grid(rows, (int)cols), fp8::ROW_THREADS, 0, s, (const T*)x, (long long)ld, (uint8_t*)q, (uint8_t*)scale,
                               (long long)rows, (int)cols, vec);
    const long long tiles = (long long)fp8::blocks_of(rows) * fp8::blocks_of(cols);
    if (tiles > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_overlapped(z ? fp8::quantize_tiles_kernel<T, true> : fp8::quantize_tiles_kernel<T, false>, (unsigned)tiles, fp8::TILE_THREADS, 0, s, (const T*)x, (long long)ld,
                             (const T*)z, (uint8_t*)q, (uint8_t*)scale, (uint8_t*)qt, (uint8_t*)scalet, sums, (int)rows, (int)cols, vec);
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
    return launch_overlapped(fp8::restore_kernel<T>, fp8::row_grid(rows, (int)cols), fp8::ROW_THREADS, 0, (cudaStream_t)stream, (const uint8_t*)q, (const uint8_t*)scale, (T*)x,
                             (long long)rows, (int)cols, fp8::whole_pieces({x}, cols, sizeof(T)));
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
    return launch_overlapped(kernel, (N + fp8::FEW_ROWS - 1) / fp8::FEW_ROWS, fp8::FEW_WARPS * 32, 0, (cudaStream_t)stream, (const T*)x, (long long)ld, (const uint8_t*)q,
                             (const uint8_t*)scale, (const T*)bias, (T*)y, tokens, N, K, gelu, fp8::whole_pieces({x}, ld, sizeof(T)));
  });
}

}  // extern "C"
