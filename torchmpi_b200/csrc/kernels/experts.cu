// Rows on their way to the experts and back: dispatch (a token's row to each of its experts' places), combine (the weighted sum of
// what the experts made of it) and their gradients.
//
// `place` (route.cu) gives the place of each entry token * k + j, `order` the entry at each place.  All passes go by tokens and read and write each
// element once.  Back to back, out of memory, bf16, 8192 x 1024: dispatch to two experts 8.5 us, 0.91 of the copy rate, to eight 26.4, 0.87; combine 12.0, 0.64, and 26.5, 0.87 (a
// thread has one piece of a row, whose loads wait for those of its places: with two experts not enough is under way).  Passes without a sum over a row give a thread one 16-byte piece of a row, so that one token of a long row is
// spread over many blocks; those with one give a warp a row.  Sums are in fp32, in one order whatever the launch: nothing is accumulated
// by atomics.  Places behind the last entry (from *used on) get zeros where the caller asks for it.
#include "act8.cuh"
#include "pdl.cuh"
#include "vec.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>

namespace tmpi {
namespace experts {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ __forceinline__ void split(long long i, int per, long long* row, int* part) {
  if ((unsigned long long)i >> 32) *row = i / per;
  else *row = (uint32_t)i / (uint32_t)per;
  *part = (int)(i - *row * per);
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d /= 2) x += __shfl_xor_sync(~0u, x, d);
  return x;
}
// zeros in the places from *used on; all threads of the grid
template <typename T, int V, int BLOCK_THREADS = THREADS>
__device__ __forceinline__ void clear_rest(const int* __restrict__ used, T* __restrict__ rows, int places, int cols) {
  if (!used) return;
  const int first = min(max(*used, 0), places);
  Pack<T, V> zero;
#pragma unroll
  for (int e = 0; e < V; ++e) zero.v[e] = from_acc<T>(0);
  const long long n = (long long)(places - first) * (cols / V);
  for (long long i = (long long)blockIdx.x * BLOCK_THREADS + threadIdx.x; i < n; i += (long long)gridDim.x * BLOCK_THREADS) st_pack<T, V>(rows + (long long)first * cols + i * V, zero);
}

// out[place of each of a token's entries] = x[token]; place_weights: the weight of the entry at each place
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) dispatch_kernel(const T* __restrict__ x, const int* __restrict__ place, const int* __restrict__ used,
                                                           const float* __restrict__ weights, T* __restrict__ out, float* __restrict__ place_weights, int places,
                                                           int tokens, int k, int cols) {
  wait_previous(x, place, used, weights);
  const int parts = cols / V;
  const long long items = (long long)tokens * parts, stride = (long long)gridDim.x * THREADS;
  constexpr int U = 2;
  for (long long i0 = (long long)blockIdx.x * THREADS + threadIdx.x; i0 < items; i0 += U * stride) {
    Pack<T, V> v[U];
    long long t[U];
    int part[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      t[u] = -1;
      if (i0 + u * stride < items) {
        split(i0 + u * stride, parts, &t[u], &part[u]);
        v[u] = ld_pack<T, V>(x + t[u] * cols + part[u] * V);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t[u] >= 0)
        for (int j = 0; j < k; ++j) {
          const int s = place[t[u] * k + j];
          if (s < 0 || s >= places) continue;
          st_pack<T, V>(out + (long long)s * cols + part[u] * V, v[u]);
          if (place_weights && part[u] == 0) place_weights[s] = weights[t[u] * k + j];
        }
  }
  clear_rest<T, V>(used, out, places, cols);
}

// The same for bf16 rows of a multiple of 8 columns, with the 8-bit checkpoint of x beside it: four threads hold the 32 elements of a block.
__global__ void __launch_bounds__(THREADS) dispatch_keep_kernel(const __nv_bfloat16* __restrict__ x, const int* __restrict__ place, __nv_bfloat16* __restrict__ out,
                                                                uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int places, int tokens, int k, int cols) {
  wait_previous(x, place);
  const int blocks = (cols + act8::BLOCK - 1) / act8::BLOCK, parts = blocks * (act8::BLOCK / 8);      // the last block of a row padded
  const long long items = (long long)tokens * parts, stride = (long long)gridDim.x * THREADS;
  for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; (i & ~31LL) < items; i += stride) {
    long long t = 0;
    int part = parts;
    if (i < items) split(i, parts, &t, &part);
    const bool in = part * 8 < cols;
    const uint4 v = in ? *reinterpret_cast<const uint4*>(x + t * cols + part * 8) : make_uint4(0u, 0u, 0u, 0u);
    if (in)
      for (int j = 0; j < k; ++j) {
        const int s = place[t * k + j];
        if (s >= 0 && s < places) *reinterpret_cast<uint4*>(out + (long long)s * cols + part * 8) = v;
      }
    const uint32_t b[4] = {v.x, v.y, v.z, v.w};
    float f[8];
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(b[e] << 16);
      f[2 * e + 1] = __uint_as_float(b[e] & 0xffff0000u);
      a = max(a, max(act8::magnitude(f[2 * e]), act8::magnitude(f[2 * e + 1])));
    }
    a = max(a, __shfl_xor_sync(~0u, a, 1));
    a = max(a, __shfl_xor_sync(~0u, a, 2));
    const uint32_t byte = act8::scale_byte(a);
    if (in) *reinterpret_cast<uint2*>(q + t * cols + part * 8) = act8::pack8(f, act8::inverse(byte));
    if (i < items && (part & 3) == 0) scale[t * blocks + part / 4] = (uint8_t)byte;
  }
}

// The dispatch of what an 8-bit checkpoint of x stands for, bf16 rows of a multiple of 8 columns.  A thread restores eight elements.
__global__ void __launch_bounds__(THREADS) dispatch8_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, const int* __restrict__ place,
                                                            __nv_bfloat16* __restrict__ out, int places, int tokens, int k, int cols) {
  wait_previous(q, scale, place);
  const int parts = cols / 8, blocks = (cols + act8::BLOCK - 1) / act8::BLOCK;
  const long long items = (long long)tokens * parts, stride = (long long)gridDim.x * THREADS;
  constexpr int U = 2;
  for (long long i0 = (long long)blockIdx.x * THREADS + threadIdx.x; i0 < items; i0 += U * stride) {
    uint2 v[U];
    uint32_t s[U];
    long long t[U];
    int part[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      t[u] = -1;
      if (i0 + u * stride >= items) continue;
      split(i0 + u * stride, parts, &t[u], &part[u]);
      v[u] = *reinterpret_cast<const uint2*>(q + t[u] * cols + part[u] * 8);
      s[u] = scale[t[u] * blocks + (part[u] >> 2)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t[u] < 0) continue;
      float f[8];
      act8::unpack8(v[u], act8::value(s[u]), f);
      Pack<__nv_bfloat16, 8> o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = __float2bfloat16_rn(f[e]);
      for (int j = 0; j < k; ++j) {
        const int at = place[t[u] * k + j];
        if (at >= 0 && at < places) st_pack<__nv_bfloat16, 8>(out + (long long)at * cols + part[u] * 8, o);
      }
    }
  }
}

// y[t] = sum over j of weights[t, j] rows[place[t, j]], added in the order of j and rounded once; weights null: ones.  An entry without a
// place adds its weight times zero: nothing, or NaN where the weight is.
template <typename R, typename T, int V, bool SLICES>
__global__ void __launch_bounds__(THREADS) combine_kernel(const R* __restrict__ rows, const float* __restrict__ weights, const int* __restrict__ place,
                                                          T* __restrict__ y, int tokens, int places, int k, int cols, int slices) {
  wait_previous(rows, weights, place);
  const int parts = cols / V;
  const long long items = (long long)tokens * parts, stride = (long long)gridDim.x * THREADS;
  for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < items; i += stride) {
    long long t;
    int part;
    split(i, parts, &t, &part);
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    constexpr int U = 4;                                  // entries in flight
    for (int j0 = 0; j0 < k; j0 += U) {
      Pack<R, V> v[U];
      float w[U];
      int s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = j0 + u < k ? place[t * k + j0 + u] : -1;
        w[u] = j0 + u < k ? weights ? weights[t * k + j0 + u] : 1.f : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if ((unsigned)s[u] < (unsigned)places) v[u] = ld_pack<R, V>(rows + (long long)s[u] * cols + part * V);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool there = (unsigned)s[u] < (unsigned)places;
        if (SLICES && there)                              // in their order
          for (int i = 1; i < slices; ++i) {
            const Pack<R, V> more = ld_pack<R, V>(rows + ((long long)i * places + s[u]) * cols + part * V);
#pragma unroll
            for (int e = 0; e < V; ++e) v[u].v[e] = from_acc<R>(to_acc<R>(v[u].v[e]) + to_acc<R>(more.v[e]));
          }
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += w[u] * (there ? (float)to_acc<R>(v[u].v[e]) : 0.f);
      }
    }
    Pack<T, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = from_acc<T>((typename AccOf<T>::type)sum[e]);
    st_pack<T, V>(y + t * cols + part * V, o);
  }
}

// The gradients of combine: drows[place] = weight dy[token], and dweights[entry] = dy[token] . rows[place] (0 for entries without a place).
// `group` threads (a power of two) share a token, a piece of its row each where there are enough of them, so that all that a token needs is under way
// at once.
constexpr int GRAD_THREADS = 128;
template <typename T, int V>
__global__ void __launch_bounds__(GRAD_THREADS) combine_gradient_kernel(const T* __restrict__ dy, const T* __restrict__ rows, const float* __restrict__ weights,
                                                                        const int* __restrict__ place, const int* __restrict__ used, T* __restrict__ drows,
                                                                        float* __restrict__ dweights, int places, int tokens, int k, int cols, int group) {
  wait_previous(dy, rows, weights, place, used);
  constexpr int J = 2;                                    // entries at a time
  __shared__ float sums[GRAD_THREADS / 32][J];
  const int lane = threadIdx.x % group, mine = threadIdx.x / group, per_block = GRAD_THREADS / group, parts = cols / V;
  const bool across = group > 32;                         // a token's sums cross warps
  for (long long t0 = (long long)blockIdx.x * per_block; t0 < tokens; t0 += (long long)gridDim.x * per_block) {      // the same for the whole block
    const long long t = t0 + mine;
    const bool in = t < tokens;
    for (int j0 = 0; j0 < k; j0 += J) {
      int s[J];
      float w[J], dot[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const bool there = in && j0 + j < k;
        s[j] = there ? place[t * k + j0 + j] : -1;
        w[j] = there ? weights[t * k + j0 + j] : 0.f;
        dot[j] = 0.f;
      }
      if (in)
        for (int c = lane; c < parts; c += group) {
          const Pack<T, V> g = ld_pack<T, V>(dy + t * cols + (long long)c * V);
          Pack<T, V> b[J];
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (rows && (unsigned)s[j] < (unsigned)places) b[j] = ld_pack<T, V>(rows + (long long)s[j] * cols + (long long)c * V);
#pragma unroll
          for (int j = 0; j < J; ++j) {
            if ((unsigned)s[j] >= (unsigned)places) continue;
            Pack<T, V> out;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float f = (float)to_acc<T>(g.v[i]);
              if (rows) dot[j] += f * (float)to_acc<T>(b[j].v[i]);
              out.v[i] = from_acc<T>((typename AccOf<T>::type)(w[j] * f));
            }
            st_pack<T, V>(drows + (long long)s[j] * cols + (long long)c * V, out);
          }
        }
      if (rows) {
        for (int d = min(group, 32) / 2; d; d /= 2)
#pragma unroll
          for (int j = 0; j < J; ++j) dot[j] += __shfl_xor_sync(~0u, dot[j], d);
        if (across) {
          if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int j = 0; j < J; ++j) sums[threadIdx.x / 32][j] = dot[j];
          __syncthreads();
          if (lane == 0)
            for (int i = 1; i < group / 32; ++i)
#pragma unroll
              for (int j = 0; j < J; ++j) dot[j] += sums[threadIdx.x / 32 + i][j];
          __syncthreads();
        }
        if (lane == 0 && in)
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (j0 + j < k) dweights[t * k + j0 + j] = (unsigned)s[j] < (unsigned)places ? dot[j] : 0.f;
      }
    }
  }
  clear_rest<T, V, GRAD_THREADS>(used, drows, places, cols);
}

// The weights' gradient in a layer of experts, a warp to a token: dweights[entry] = the sum of the entry's place over `dots` (four slices side by side,
// grouped.cu) + dy[token] . bias[expert]; 0 for entries without a place.  By tokens, what belongs to the entries and the row of dy are one step of
// loads, and the row is read once; two entries at a time, the slices of each by half a warp.  8192 x 1024 and two
// experts of eight 9.8 us, eight of 64 27.5; 12.8 and 34.2 where each slice lay apart (a lane to a slice: a load touched 32 lines).
template <int V>
__global__ void __launch_bounds__(THREADS) weight_gradient_kernel(const float* __restrict__ dots, const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ bias,
                                                                  const int* __restrict__ place, const int* __restrict__ chosen, float* __restrict__ dweights,
                                                                  int places, int tokens, int k, int slices, int cols, int nexperts) {
  wait_previous(dots, dy, bias, place, chosen);
  const int lane = threadIdx.x & 31, parts = cols / V;
  for (long long t = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); t < tokens; t += (long long)gridDim.x * WARPS) {
    constexpr int J = 2, U = 4;
    for (int j0 = 0; j0 < k; j0 += J) {
      const int js = j0 + (lane >> 4);                    // the entry whose slices this lane adds
      const int s = js < k ? place[t * k + js] : -1;
      int e[J];
      float sum[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        e[j] = j0 + j < k && bias ? chosen[t * k + j0 + j] : -1;
        sum[j] = 0.f;
      }
      const bool there = (unsigned)s < (unsigned)places;
      float of_slices = 0.f;
      if (there)
#pragma unroll 2
        for (int i = lane & 15; 4 * i < slices; i += 16) {
          const float4 v = *reinterpret_cast<const float4*>(dots + ((long long)i * places + s) * 4);
          of_slices += v.x + (4 * i + 1 < slices ? v.y : 0.f) + (4 * i + 2 < slices ? v.z : 0.f) + (4 * i + 3 < slices ? v.w : 0.f);
        }
      if (bias)
        for (int c0 = lane; c0 < parts; c0 += 32 * U) {
          Pack<__nv_bfloat16, V> g[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + 32 * u < parts) g[u] = ld_pack<__nv_bfloat16, V>(dy + t * cols + (long long)(c0 + 32 * u) * V);
#pragma unroll
          for (int j = 0; j < J; ++j) {
            if ((unsigned)e[j] >= (unsigned)nexperts) continue;
            Pack<__nv_bfloat16, V> b[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (c0 + 32 * u < parts) b[u] = ld_pack<__nv_bfloat16, V>(bias + (long long)e[j] * cols + (long long)(c0 + 32 * u) * V);
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (c0 + 32 * u < parts)
#pragma unroll
                for (int i = 0; i < V; ++i) sum[j] += __bfloat162float(g[u].v[i]) * __bfloat162float(b[u].v[i]);
          }
        }
#pragma unroll
      for (int d = 8; d; d /= 2) of_slices += __shfl_xor_sync(~0u, of_slices, d);
#pragma unroll
      for (int j = 0; j < J; ++j) sum[j] = warp_sum(sum[j]);
      if ((lane & 15) == 0 && js < k) dweights[t * k + js] = there ? of_slices + (lane ? sum[1] : sum[0]) : 0.f;
    }
  }
}

static int grid_items(long long items, int u, int per_sm) {
  return (int)std::max<long long>(1, std::min<long long>((items + THREADS * u - 1) / (THREADS * u), 148LL * per_sm));
}
static int grid_rows(int rows, int per_sm) { return std::max(1, std::min((rows + WARPS - 1) / WARPS, 148 * per_sm)); }

// f(element type, elements of a piece): 16-byte pieces where rows are whole ones and all tensors start on such a boundary, else single elements
template <typename F>
static cudaError_t by_type(int dtype, int cols, std::initializer_list<const void*> tensors, F f) {
  const bool wide = all_aligned16(tensors);
  auto with = [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    return wide && cols % V == 0 ? f(t, std::integral_constant<int, V>()) : f(t, std::integral_constant<int, 1>());
  };
  if (dtype == TMPI_BF16) return with(__nv_bfloat16());
  if (dtype == TMPI_F16) return with(__half());
  return with(float());
}

static int checked(int tokens, int k, int cols, int dtype, const char* what) {
  if (tokens < 0 || k < 1 || cols < 1 || (long long)tokens * k > 1LL << 30) return fail(TMPI_ERR_INVALID, "%s: %d tokens of %d experts, rows of %d", what, tokens, k, cols);
  if (dtype != TMPI_BF16 && dtype != TMPI_F16 && dtype != TMPI_F32) return fail(TMPI_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  return TMPI_OK;
}
static int finish(cudaError_t e, const char* what) {
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace experts
}  // namespace tmpi

using namespace tmpi;

extern "C" {

// out [tokens * k, cols] from x [tokens, cols]; used (optional): places from *used on get zeros; place_weights [tokens * k] (optional): the
// weights [tokens, k] in the order of the places
int tmpi_expert_dispatch(const void* x, const int* place, const int* used, const float* weights, void* out, float* place_weights, int tokens, int k, int cols, int dtype, void* stream) {
  const int st = experts::checked(tokens, k, cols, dtype, "expert_dispatch");
  if (st || !tokens) return st;
  return experts::finish(experts::by_type(dtype, cols, {x, out}, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    return launch_overlapped(experts::dispatch_kernel<T, V>, experts::grid_items((long long)tokens * (cols / V), 2, 8), experts::THREADS, 0, (cudaStream_t)stream,
                             (const T*)x, place, used, weights, (T*)out, place_weights, tokens * k, tokens, k, cols);
  }), "expert_dispatch");
}

// The same for bf16, and x's 8-bit checkpoint in q [tokens, cols], scale [tokens, ceil(cols / 32)]; cols a multiple of 8, 16-byte boundaries
int tmpi_expert_dispatch_keep(const void* x, const int* place, void* out, void* q, void* scale, int tokens, int k, int cols, void* stream) {
  const int st = experts::checked(tokens, k, cols, TMPI_BF16, "expert_dispatch_keep");
  if (st || !tokens) return st;
  if (cols % 8 || !all_aligned16({x, out}) || ((uintptr_t)q & 7)) return fail(TMPI_ERR_INVALID, "expert_dispatch_keep: rows must be multiples of 16 bytes, on 16-byte boundaries");
  const long long items = (long long)tokens * ((cols + 31) / 32) * 4;
  return experts::finish(launch_overlapped(experts::dispatch_keep_kernel, experts::grid_items(items, 1, 8), experts::THREADS, 0, (cudaStream_t)stream,
                                           (const __nv_bfloat16*)x, place, (__nv_bfloat16*)out, (uint8_t*)q, (uint8_t*)scale, tokens * k, tokens, k, cols),
                         "expert_dispatch_keep");
}

// out [tokens * k, cols] bf16 from the 8-bit checkpoint of x; cols a multiple of 8
int tmpi_expert_dispatch8(const void* q, const void* scale, const int* place, void* out, int tokens, int k, int cols, void* stream) {
  const int st = experts::checked(tokens, k, cols, TMPI_BF16, "expert_dispatch8");
  if (st || !tokens) return st;
  if (cols % 8 || ((uintptr_t)q & 7) || !all_aligned16({out})) return fail(TMPI_ERR_INVALID, "expert_dispatch8: rows must be multiples of 16 bytes, on 16-byte boundaries");
  return experts::finish(launch_overlapped(experts::dispatch8_kernel, experts::grid_items((long long)tokens * (cols / 8), 2, 8), experts::THREADS, 0, (cudaStream_t)stream,
                                           (const uint8_t*)q, (const uint8_t*)scale, place, (__nv_bfloat16*)out, tokens * k, tokens, k, cols), "expert_dispatch8");
}

// y [tokens, cols] of `dtype` from rows [tokens * k, cols] of `dtype`, or (fp32_slices > 0, y bf16) from the sum of fp32 rows [slices, tokens * k, cols];
// weights [tokens, k] or null
int tmpi_expert_combine(const void* rows, int fp32_slices, const float* weights, const int* place, void* y, int tokens, int k, int cols, int dtype, void* stream) {
  const int st = experts::checked(tokens, k, cols, dtype, "expert_combine");
  if (st || !tokens) return st;
  if (fp32_slices < 0) return fail(TMPI_ERR_INVALID, "expert_combine: %d slices", fp32_slices);
  if (fp32_slices && dtype != TMPI_BF16) return fail(TMPI_ERR_UNSUPPORTED, "expert_combine: fp32 rows to dtype %d", dtype);
  auto go = [&](auto r, auto t, auto v) {
    using R = decltype(r);
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const auto kernel = fp32_slices > 1 ? experts::combine_kernel<R, T, V, sizeof(R) == 4> : experts::combine_kernel<R, T, V, false>;
    return launch_overlapped(kernel, experts::grid_items((long long)tokens * (cols / V), 1, 8), experts::THREADS, 0, (cudaStream_t)stream, (const R*)rows, weights,
                             place, (T*)y, tokens, tokens * k, k, cols, std::max(1, fp32_slices));
  };
  if (fp32_slices) {
    const bool wide = cols % 8 == 0 && (uintptr_t)rows % 32 == 0 && all_aligned16({y});
    return experts::finish(wide ? go(float(), __nv_bfloat16(), std::integral_constant<int, 8>()) : go(float(), __nv_bfloat16(), std::integral_constant<int, 1>()),
                           "expert_combine");
  }
  return experts::finish(experts::by_type(dtype, cols, {rows, y}, [&](auto t, auto v) { return go(t, t, v); }), "expert_combine");
}

// drows [tokens * k, cols] = weight times dy [tokens, cols], zeros from *used on, and, where rows [tokens * k, cols] is given, dweights [tokens * k]
int tmpi_expert_combine_gradient(const void* dy, const void* rows, const float* weights, const int* place, const int* used, void* drows, float* dweights, int tokens,
                                 int k, int cols, int dtype, void* stream) {
  const int st = experts::checked(tokens, k, cols, dtype, "expert_combine_gradient");
  if (st || !tokens) return st;
  if (rows && !dweights) return fail(TMPI_ERR_INVALID, "expert_combine_gradient: rows without dweights");
  return experts::finish(experts::by_type(dtype, cols, {dy, rows, drows}, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    int group = 1;
    while (group < experts::GRAD_THREADS && group < cols / V) group *= 2;
    const int per_block = experts::GRAD_THREADS / group, blocks = std::min((tokens + per_block - 1) / per_block, 148 * 16);
    return launch_overlapped(experts::combine_gradient_kernel<T, V>, blocks, experts::GRAD_THREADS, 0, (cudaStream_t)stream, (const T*)dy, (const T*)rows, weights,
                             place, used, (T*)drows, dweights, tokens * k, tokens, k, cols, group);
  }), "expert_combine_gradient");
}

// dweights [tokens, k] = the sums over dots [ceil(slices / 4), tokens * k, 4] of the entries' places + dy [tokens, cols] . bias [nexperts, cols] (bf16, or null) of
// the chosen expert
int tmpi_expert_weight_gradient(const float* dots, const void* dy, const void* bias, const int* place, const int* chosen, float* dweights, int tokens, int k,
                                int slices, int cols, int nexperts, void* stream) {
  const int st = experts::checked(tokens, k, cols, TMPI_BF16, "expert_weight_gradient");
  if (st || !tokens) return st;
  if ((uintptr_t)dots & 15) return fail(TMPI_ERR_INVALID, "expert_weight_gradient: dots must be 16-byte aligned");
  const auto kernel = cols % 8 == 0 && all_aligned16({dy, bias}) ? experts::weight_gradient_kernel<8> : experts::weight_gradient_kernel<1>;
  return experts::finish(launch_overlapped(kernel, experts::grid_rows(tokens, 8), experts::THREADS, 0, (cudaStream_t)stream, dots, (const __nv_bfloat16*)dy,
                                           (const __nv_bfloat16*)bias, place, chosen, dweights, tokens * k, tokens, k, slices, cols, nexperts), "expert_weight_gradient");
}

}  // extern "C"
