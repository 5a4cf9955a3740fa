// 8-bit activation checkpoints (act8.cuh has the format): quantize, restore, and the GELU backward that reads one.
//
// Every element is read and written once.  Four threads hold the 32 elements of a block, eight each, so a block's
// largest magnitude takes two shuffles, loads are 16 bytes and more per thread and a warp's loads are consecutive.  Rows whose length
// is no multiple of 8 elements, or that do not start on a 16-byte boundary, take the same kernels with single elements (VEC = false).
// With whole pieces they are bound by memory.  Measured, bf16, us and share of the copy rate: 65536 x 4096 quantize 145 (0.86), restore 137 (0.91), GELU backward 317 (0.91) after a flush of the L2;
// 32768 x 1024 back to back 19.5 and 15.9, in one wave of blocks that loop (two waves: 21.4 and 17.3; 65536 x 4096 is the same either way).
// Single elements are bound by their loads and stores, a byte or two of each: 32768 x 1001, after a flush, quantize 51, restore 98, GELU backward 169, where 1000
// columns take 38, 24 and 57.
#include "act8.cuh"
#include "gelu.cuh"
#include "pdl.cuh"
#include "vec.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>

namespace tmpi {
namespace act8 {

constexpr int THREADS = 256;
constexpr int PER = 8;                    // elements of a thread

// Where the eight elements of work item i lie: four items per block, the last block of a row padded.
struct Place { long long row; int col; };
struct Layout {
  long long rows;
  int cols, blocks;                       // blocks: of a row
  int linear;                             // rows follow each other in whole blocks: item i starts at element 8 i
  __device__ __forceinline__ long long items() const { return rows * blocks * (BLOCK / PER); }
  __device__ __forceinline__ long long at(long long i) const {          // first element
    if (linear) return i * PER;
    const Place p = place(i);
    return p.row * cols + p.col;
  }
  __device__ __forceinline__ Place place(long long i) const {
    const int per_row = blocks * (BLOCK / PER);
    long long row;
    if ((unsigned long long)i >> 32) row = i / per_row;
    else row = (uint32_t)i / (uint32_t)per_row;
    return {row, (int)(i - row * per_row) * PER};
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, float (&x)[PER]) {      // n: elements of the item inside its row
  if (VEC) {
    constexpr int V = 16 / sizeof(T);
    if (n > 0) {
#pragma unroll
      for (int j = 0; j < PER / V; ++j) {
        const Pack<T, V> a = ld_pack<T, V>(p + j * V);
#pragma unroll
        for (int k = 0; k < V; ++k) x[j * V + k] = (float)to_acc<T>(a.v[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k) x[k] = 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = k < n ? (float)to_acc<T>(p[k]) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&x)[PER]) {
  if (VEC) {
    constexpr int V = 16 / sizeof(T);
    if (n <= 0) return;
#pragma unroll
    for (int j = 0; j < PER / V; ++j) {
      Pack<T, V> a;
#pragma unroll
      for (int k = 0; k < V; ++k) a.v[k] = from_acc<T>((typename AccOf<T>::type)x[j * V + k]);
      st_pack<T, V>(p + j * V, a);
    }
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (k < n) p[k] = from_acc<T>((typename AccOf<T>::type)x[k]);
  }
}
template <bool VEC>
__device__ __forceinline__ uint2 load_q(const uint8_t* __restrict__ p, int n) {
  if (VEC) return n > 0 ? *reinterpret_cast<const uint2*>(p) : make_uint2(0u, 0u);
  uint2 q = make_uint2(0u, 0u);
#pragma unroll
  for (int k = 0; k < PER; ++k)
    if (k < n) (k < 4 ? q.x : q.y) |= (uint32_t)p[k] << (8 * (k & 3));
  return q;
}
template <bool VEC>
__device__ __forceinline__ void store_q(uint8_t* __restrict__ p, int n, uint2 q) {
  if (VEC) {
    if (n > 0) *reinterpret_cast<uint2*>(p) = q;
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (k < n) p[k] = (uint8_t)((k < 4 ? q.x : q.y) >> (8 * (k & 3)));
  }
}

// Items U apart are in flight together.  The threads of a warp stay together (the loop's bound is rounded up to whole warps), for the shuffles.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ scale, const Layout l) {
  wait_previous(x);
  const long long items = l.items(), stride = (long long)gridDim.x * THREADS;
  constexpr int U = 16 / sizeof(T) / 2;                 // 64 bytes of a thread
  for (long long i0 = (long long)blockIdx.x * THREADS + threadIdx.x; (i0 & ~31LL) < items; i0 += U * stride) {
    float v[U][PER];
    int n[U];
    long long at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * stride;
      n[u] = 0;
      at[u] = 0;
      if (i < items) {
        at[u] = l.at(i);
        n[u] = l.linear ? PER : l.cols - l.place(i).col;
      }
      load8<T, VEC>(x + at[u], n[u], v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t a = 0;                                   // largest magnitude, infinities and NaN among them: they are looked at where a warp has one
#pragma unroll
      for (int k = 0; k < PER; ++k) a = max(a, __float_as_uint(v[u][k]) & 0x7fffffffu);
      const bool finite = __all_sync(~0u, a < 0x7f800000u);
      if (!finite) {
        a = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) a = max(a, magnitude(v[u][k]));
      }
      a = max(a, __shfl_xor_sync(~0u, a, 1));
      a = max(a, __shfl_xor_sync(~0u, a, 2));
      const uint32_t byte = scale_byte(a);
      const long long i = i0 + u * stride;
      store_q<VEC>(q + at[u], n[u], finite ? pack8_finite(v[u], inverse(byte)) : pack8(v[u], inverse(byte)));
      if ((threadIdx.x & 3) == 0 && i < items) scale[i >> 2] = (uint8_t)byte;
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) restore_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, T* __restrict__ x, const Layout l) {
  wait_previous(q, scale);
  const long long items = l.items(), stride = (long long)gridDim.x * THREADS;
  constexpr int U = 4;
  for (long long i0 = (long long)blockIdx.x * THREADS + threadIdx.x; i0 < items; i0 += U * stride) {
    uint2 v[U];
    uint32_t s[U];
    int n[U];
    long long at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * stride;
      n[u] = 0;
      at[u] = 0;
      s[u] = 0;
      if (i < items) {
        at[u] = l.at(i);
        n[u] = l.linear ? PER : l.cols - l.place(i).col;
        s[u] = scale[i >> 2];
      }
      v[u] = load_q<VEC>(q + at[u], n[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[PER];
      unpack8(v[u], value(s[u]), f);
      store8<T, VEC>(x + at[u], n[u], f);
    }
  }
}

// dz = dy gelu'(z~), h = gelu(z~) for the checkpoint z~ of z.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS, 4) gelu_gradient_kernel(const T* __restrict__ dy, const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                                   T* __restrict__ dz, T* __restrict__ h, const Layout l) {
  wait_previous(dy, q, scale);
  const long long items = l.items(), stride = (long long)gridDim.x * THREADS;
  constexpr int U = 2;
  for (long long i0 = (long long)blockIdx.x * THREADS + threadIdx.x; i0 < items; i0 += U * stride) {
    float g[U][PER];
    uint2 v[U];
    uint32_t s[U];
    int n[U];
    long long at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * stride;
      n[u] = 0;
      at[u] = 0;
      s[u] = 0;
      if (i < items) {
        at[u] = l.at(i);
        n[u] = l.linear ? PER : l.cols - l.place(i).col;
        s[u] = scale[i >> 2];
      }
      v[u] = load_q<VEC>(q + at[u], n[u]);
      load8<T, VEC>(dy + at[u], n[u], g[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float z[PER], y[PER];
      unpack8(v[u], value(s[u]), z);
#pragma unroll
      for (int k = 0; k < PER; k += 2) {
        float d0, d1;
        if (sizeof(T) == 2) {                           // results of 8 or 11 bits: the quicker form (gelu.cuh)
          unsigned long long value2, slope2;
          quick_gelu_both2(attn_util::pack2(__float_as_uint(z[k]), __float_as_uint(z[k + 1])), &value2, &slope2);
          attn_util::unpack2(value2, y[k], y[k + 1]);
          attn_util::unpack2(slope2, d0, d1);
        } else {
          gelu_both2(z[k], z[k + 1], &y[k], &y[k + 1], &d0, &d1);
        }
        g[u][k] *= d0;
        g[u][k + 1] *= d1;
      }
      store8<T, VEC>(dz + at[u], n[u], g[u]);
      if (h) store8<T, VEC>(h + at[u], n[u], y);
    }
  }
}

static Layout layout(int64_t rows, int cols) {
  Layout l;
  l.rows = rows;
  l.cols = cols;
  l.blocks = (cols + BLOCK - 1) / BLOCK;
  l.linear = cols % BLOCK == 0;
  return l;
}
// blocks of a launch for items that a thread takes `u` at a time
static int grid(const Layout& l, int u, int per_sm) {
  const long long items = l.rows * l.blocks * (BLOCK / PER);
  return (int)std::min<long long>((items + THREADS * u - 1) / (THREADS * u), 148LL * per_sm);
}
static bool vectors(int cols, std::initializer_list<const void*> wide, const void* q) {
  return cols % PER == 0 && all_aligned16(wide) && !((uintptr_t)q & 7);
}

template <typename T>
static cudaError_t quantize_t(const void* x, void* q, void* scale, const Layout& l, cudaStream_t s) {
  const auto kernel = vectors(l.cols, {x}, q) ? quantize_kernel<T, true> : quantize_kernel<T, false>;
  return launch_overlapped(kernel, grid(l, 16 / sizeof(T) / 2, 4), THREADS, 0, s, (const T*)x, (uint8_t*)q, (uint8_t*)scale, l);
}
template <typename T>
static cudaError_t restore_t(const void* q, const void* scale, void* x, const Layout& l, cudaStream_t s) {
  const auto kernel = vectors(l.cols, {x}, q) ? restore_kernel<T, true> : restore_kernel<T, false>;
  return launch_overlapped(kernel, grid(l, 4, 4), THREADS, 0, s, (const uint8_t*)q, (const uint8_t*)scale, (T*)x, l);
}
template <typename T>
static cudaError_t gelu_gradient_t(const void* dy, const void* q, const void* scale, void* dz, void* h, const Layout& l, cudaStream_t s) {
  const auto kernel = vectors(l.cols, {dy, dz, h}, q) ? gelu_gradient_kernel<T, true> : gelu_gradient_kernel<T, false>;
  return launch_overlapped(kernel, grid(l, 2, 4), THREADS, 0, s, (const T*)dy, (const uint8_t*)q, (const uint8_t*)scale, (T*)dz, (T*)h, l);
}

static int finish(cudaError_t e, const char* what) {
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}
static int checked(int64_t rows, int cols, const char* what) {
  if (rows < 0 || cols < 1 || rows > (int64_t)1 << 40) return fail(TMPI_ERR_INVALID, "%s: %lld rows of %d", what, (long long)rows, cols);
  return TMPI_OK;
}

}  // namespace act8
}  // namespace tmpi

using namespace tmpi;

extern "C" {

// x [rows, cols] of `dtype` -> q [rows, cols] e4m3, scale [rows, ceil(cols / 32)]
int tmpi_act8_quantize(const void* x, void* q, void* scale, int64_t rows, int cols, int dtype, void* stream) {
  const int st = act8::checked(rows, cols, "act8_quantize");
  if (st || !rows) return st;
  const act8::Layout l = act8::layout(rows, cols);
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case TMPI_BF16: return act8::finish(act8::quantize_t<__nv_bfloat16>(x, q, scale, l, s), "act8_quantize");
    case TMPI_F16: return act8::finish(act8::quantize_t<__half>(x, q, scale, l, s), "act8_quantize");
    case TMPI_F32: return act8::finish(act8::quantize_t<float>(x, q, scale, l, s), "act8_quantize");
  }
  return fail(TMPI_ERR_UNSUPPORTED, "act8_quantize: dtype %d", dtype);
}

int tmpi_act8_restore(const void* q, const void* scale, void* x, int64_t rows, int cols, int dtype, void* stream) {
  const int st = act8::checked(rows, cols, "act8_restore");
  if (st || !rows) return st;
  const act8::Layout l = act8::layout(rows, cols);
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case TMPI_BF16: return act8::finish(act8::restore_t<__nv_bfloat16>(q, scale, x, l, s), "act8_restore");
    case TMPI_F16: return act8::finish(act8::restore_t<__half>(q, scale, x, l, s), "act8_restore");
    case TMPI_F32: return act8::finish(act8::restore_t<float>(q, scale, x, l, s), "act8_restore");
  }
  return fail(TMPI_ERR_UNSUPPORTED, "act8_restore: dtype %d", dtype);
}

// dz = dy gelu'(z~) and, where h is given, h = gelu(z~), all [rows, cols] of `dtype`, for the checkpoint (q, scale) z~ of z
int tmpi_act8_gelu_gradient(const void* dy, const void* q, const void* scale, void* dz, void* h, int64_t rows, int cols, int dtype, void* stream) {
  const int st = act8::checked(rows, cols, "act8_gelu_gradient");
  if (st || !rows) return st;
  const act8::Layout l = act8::layout(rows, cols);
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case TMPI_BF16: return act8::finish(act8::gelu_gradient_t<__nv_bfloat16>(dy, q, scale, dz, h, l, s), "act8_gelu_gradient");
    case TMPI_F16: return act8::finish(act8::gelu_gradient_t<__half>(dy, q, scale, dz, h, l, s), "act8_gelu_gradient");
    case TMPI_F32: return act8::finish(act8::gelu_gradient_t<float>(dy, q, scale, dz, h, l, s), "act8_gelu_gradient");
  }
  return fail(TMPI_ERR_UNSUPPORTED, "act8_gelu_gradient: dtype %d", dtype);
}

}  // extern "C"
