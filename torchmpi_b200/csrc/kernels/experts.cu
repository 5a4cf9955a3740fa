// Rows on their way to the experts and back: dispatch (a token's row to each of its experts' places), combine (the weighted sum of
// what the experts made of it) and their gradients.
//
// `order` (route.cu) gives the entry token * k + j at each place, `place` the place of each entry.  All passes read and write each element once
// and are bound by memory.  Passes without a sum over a row give a thread one 16-byte piece of a row, so that one token of a long row is
// spread over many blocks; those with one give a warp a row.  Sums are in fp32, in one order whatever the launch: nothing is accumulated
// by atomics.
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
// the token of the entry at place `s`, -1 for places that hold none; entries that no token has (a caller's own order) count as none
__device__ __forceinline__ int token_at(const int* __restrict__ order, int s, int k, int tokens) {
  const int e = order[s];
  return e >= 0 && e / k < tokens ? e / k : -1;
}

// out[s] = x[token of s], zeros where there is none
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) dispatch_kernel(const T* __restrict__ x, const int* __restrict__ order, T* __restrict__ out, int places, int tokens,
                                                           int k, int cols) {
  wait_previous(x, order);
  const int parts = cols / V;
  const long long items = (long long)places * parts, stride = (long long)gridDim.x * THREADS;
  constexpr int U = 4;
  for (long long i0 = (long long)blockIdx.x * THREADS + threadIdx.x; i0 < items; i0 += U * stride) {
    Pack<T, V> v[U];
    long long row[U];
    int part[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * stride;
      if (i >= items) { row[u] = -1; continue; }
      split(i, parts, &row[u], &part[u]);
      const int t = token_at(order, (int)row[u], k, tokens);
      if (t >= 0) {
        v[u] = ld_pack<T, V>(x + (long long)t * cols + part[u] * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[u].v[e] = from_acc<T>(0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] >= 0) st_pack<T, V>(out + row[u] * cols + part[u] * V, v[u]);
  }
}

// The same from the 8-bit checkpoint of x, in bf16.  A thread restores eight elements.
template <bool VEC>
__global__ void __launch_bounds__(THREADS) dispatch8_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, const int* __restrict__ order,
                                                            __nv_bfloat16* __restrict__ out, int places, int tokens, int k, int cols) {
  wait_previous(q, scale, order);
  const int parts = (cols + 7) / 8, blocks = (cols + act8::BLOCK - 1) / act8::BLOCK;
  const long long items = (long long)places * parts, stride = (long long)gridDim.x * THREADS;
  constexpr int U = 4;
  for (long long i0 = (long long)blockIdx.x * THREADS + threadIdx.x; i0 < items; i0 += U * stride) {
    uint2 v[U];
    uint32_t s[U];
    long long row[U];
    int part[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * stride;
      row[u] = -1;
      part[u] = 0;
      v[u] = make_uint2(0u, 0u);
      s[u] = 1;
      if (i >= items) continue;
      split(i, parts, &row[u], &part[u]);
      const int t = token_at(order, (int)row[u], k, tokens);
      if (t < 0) continue;
      s[u] = scale[(long long)t * blocks + (part[u] >> 2)];
      const uint8_t* from = q + (long long)t * cols + part[u] * 8;
      if (VEC) {
        v[u] = *reinterpret_cast<const uint2*>(from);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (part[u] * 8 + e < cols) (e < 4 ? v[u].x : v[u].y) |= (uint32_t)from[e] << (8 * (e & 3));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row[u] < 0) continue;
      float f[8];
      act8::unpack8(v[u], act8::value(s[u]), f);
      __nv_bfloat16* to = out + row[u] * cols + part[u] * 8;
      if (VEC) {
        Pack<__nv_bfloat16, 8> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = __float2bfloat16_rn(f[e]);
        st_pack<__nv_bfloat16, 8>(to, o);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (part[u] * 8 + e < cols) to[e] = __float2bfloat16_rn(f[e]);
      }
    }
  }
}

// y[t] = sum over j of weights[t, j] rows[place[t, j]], added in the order of j and rounded once; weights null: ones.  An entry without a
// place adds its weight times zero: nothing, or NaN where the weight is.
template <typename R, typename T, int V>
__global__ void __launch_bounds__(THREADS) combine_kernel(const R* __restrict__ rows, const float* __restrict__ weights, const int* __restrict__ place,
                                                          T* __restrict__ y, int tokens, int places, int k, int cols) {
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
      bool there[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        there[u] = false;
        w[u] = 0.f;
        if (j0 + u >= k) continue;
        const int s = place[t * k + j0 + u];
        w[u] = weights ? weights[t * k + j0 + u] : 1.f;
        there[u] = s >= 0 && s < places;
        if (there[u]) v[u] = ld_pack<R, V>(rows + (long long)s * cols + part * V);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += w[u] * (there[u] ? (float)to_acc<R>(v[u].v[e]) : 0.f);
    }
    Pack<T, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = from_acc<T>((typename AccOf<T>::type)sum[e]);
    st_pack<T, V>(y + t * cols + part * V, o);
  }
}

// The gradients of combine, a warp to a place: drows[s] = weight dy[token] (without `scaled` dy[token] itself), and
// dweights[entry] = dy[token] . other, where other is rows[s] or, with `chosen`, the row of the entry's expert (its bias).  Places without an
// entry get zeros; dweights of entries without a place are left to the caller.  place_weights: the weight of the entry at each place.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) combine_gradient_kernel(const T* __restrict__ dy, const T* __restrict__ other, const float* __restrict__ weights,
                                                                   const int* __restrict__ order, const int* __restrict__ chosen, T* __restrict__ drows,
                                                                   float* __restrict__ dweights, float* __restrict__ place_weights, int scaled,
                                                                   int places, int tokens, int k, int cols, int nexperts) {
  wait_previous(dy, other, weights, order, chosen);
  const int lane = threadIdx.x & 31, parts = cols / V;
  for (long long s = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); s < places; s += (long long)gridDim.x * WARPS) {
    const int t = token_at(order, (int)s, k, tokens), entry = t >= 0 ? order[s] : 0;
    const float w = t >= 0 && weights ? weights[entry] : 1.f;
    const T* o = other;
    if (other && t >= 0) {
      const int e = chosen ? chosen[entry] : 0;
      o = chosen ? (e >= 0 && e < nexperts ? other + (long long)e * cols : nullptr) : other + s * cols;
    }
    float dot = 0.f;
    for (int c0 = lane; c0 < parts; c0 += 4 * 32) {
      Pack<T, V> g[4], b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = c0 + 32 * u;
        if (c < parts && t >= 0) {
          g[u] = ld_pack<T, V>(dy + (long long)t * cols + c * V);
          if (o) b[u] = ld_pack<T, V>(o + (long long)c * V);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) g[u].v[e] = b[u].v[e] = from_acc<T>(0);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = c0 + 32 * u;
        if (c >= parts) break;
        Pack<T, V> out;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float f = (float)to_acc<T>(g[u].v[e]);
          if (o) dot += f * (float)to_acc<T>(b[u].v[e]);
          out.v[e] = scaled ? from_acc<T>((typename AccOf<T>::type)(w * f)) : g[u].v[e];
        }
        st_pack<T, V>(drows + s * cols + (long long)c * V, out);
      }
    }
    if (place_weights && lane == 0) place_weights[s] = t >= 0 ? w : 0.f;
    if (dweights) {
      dot = warp_sum(dot);
      if (lane == 0 && t >= 0) dweights[entry] = dot;
    }
  }
}

// dweights[entry] += the sum of the entry's row of `dots` (grouped.cu: a number for 64 columns), a warp to a place
__global__ void __launch_bounds__(THREADS) dots_kernel(const float* __restrict__ dots, const int* __restrict__ order, float* __restrict__ dweights, int places, int tokens,
                                                       int k, int slices) {
  wait_previous(dots, order);
  const int lane = threadIdx.x & 31;
  for (long long s = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); s < places; s += (long long)gridDim.x * WARPS) {
    if (token_at(order, (int)s, k, tokens) < 0) continue;
    float sum = 0.f;
    for (int i = lane; i < slices; i += 32) sum += dots[s * slices + i];
    sum = warp_sum(sum);
    if (lane == 0) dweights[order[s]] += sum;
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

// out [tokens * k, cols] from x [tokens, cols]
int tmpi_expert_dispatch(const void* x, const int* order, void* out, int tokens, int k, int cols, int dtype, void* stream) {
  const int st = experts::checked(tokens, k, cols, dtype, "expert_dispatch");
  if (st || !tokens) return st;
  const int places = tokens * k;
  return experts::finish(experts::by_type(dtype, cols, {x, out}, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    return launch_overlapped(experts::dispatch_kernel<T, V>, experts::grid_items((long long)places * (cols / V), 4, 8), experts::THREADS, 0, (cudaStream_t)stream,
                             (const T*)x, order, (T*)out, places, tokens, k, cols);
  }), "expert_dispatch");
}

// The same from an 8-bit checkpoint of x, in bf16
int tmpi_expert_dispatch8(const void* q, const void* scale, const int* order, void* out, int tokens, int k, int cols, void* stream) {
  const int st = experts::checked(tokens, k, cols, TMPI_BF16, "expert_dispatch8");
  if (st || !tokens) return st;
  const int places = tokens * k;
  const auto kernel = cols % 8 == 0 && !((uintptr_t)q & 7) && all_aligned16({out}) ? experts::dispatch8_kernel<true> : experts::dispatch8_kernel<false>;
  return experts::finish(launch_overlapped(kernel, experts::grid_items((long long)places * ((cols + 7) / 8), 4, 8), experts::THREADS, 0, (cudaStream_t)stream,
                                           (const uint8_t*)q, (const uint8_t*)scale, order, (__nv_bfloat16*)out, places, tokens, k, cols), "expert_dispatch8");
}

// y [tokens, cols] of `dtype` from rows [tokens * k, cols] of `dtype`, or in fp32 (rows_fp32: y bf16); weights [tokens, k] or null
int tmpi_expert_combine(const void* rows, int rows_fp32, const float* weights, const int* place, void* y, int tokens, int k, int cols, int dtype, void* stream) {
  const int st = experts::checked(tokens, k, cols, dtype, "expert_combine");
  if (st || !tokens) return st;
  if (rows_fp32 && dtype != TMPI_BF16) return fail(TMPI_ERR_UNSUPPORTED, "expert_combine: fp32 rows to dtype %d", dtype);
  auto go = [&](auto r, auto t, auto v) {
    using R = decltype(r);
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    return launch_overlapped(experts::combine_kernel<R, T, V>, experts::grid_items((long long)tokens * (cols / V), 1, 8), experts::THREADS, 0, (cudaStream_t)stream,
                             (const R*)rows, weights, place, (T*)y, tokens, tokens * k, k, cols);
  };
  if (rows_fp32) {
    const bool wide = cols % 4 == 0 && all_aligned16({rows, y});
    return experts::finish(wide ? go(float(), __nv_bfloat16(), std::integral_constant<int, 4>()) : go(float(), __nv_bfloat16(), std::integral_constant<int, 1>()),
                           "expert_combine");
  }
  return experts::finish(experts::by_type(dtype, cols, {rows, y}, [&](auto t, auto v) { return go(t, t, v); }), "expert_combine");
}

// drows [tokens * k, cols] and, where given, dweights [tokens * k] (of the entries that have a place) from dy [tokens, cols].  other: rows
// [tokens * k, cols], or with `chosen` a row for each of nexperts experts; null: no dweights.  scaled: drows holds weight times dy, else
// dy.  place_weights [tokens * k] (optional): the weights in the order of the places.
int tmpi_expert_combine_gradient(const void* dy, const void* other, const float* weights, int scaled, const int* order, const int* chosen, void* drows,
                                 float* dweights, float* place_weights, int tokens, int k, int cols, int nexperts, int dtype, void* stream) {
  const int st = experts::checked(tokens, k, cols, dtype, "expert_combine_gradient");
  if (st || !tokens) return st;
  if (dweights && !other) return fail(TMPI_ERR_INVALID, "expert_combine_gradient: dweights without the rows");
  return experts::finish(experts::by_type(dtype, cols, {dy, other, drows}, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    return launch_overlapped(experts::combine_gradient_kernel<T, V>, experts::grid_rows(tokens * k, 8), experts::THREADS, 0, (cudaStream_t)stream, (const T*)dy,
                             (const T*)other, weights, order, chosen, (T*)drows, dweights, place_weights, scaled, tokens * k, tokens, k, cols, nexperts);
  }), "expert_combine_gradient");
}

// dweights [tokens * k] += the sums of the rows of dots [tokens * k, slices], for the entries that have a place
int tmpi_expert_dots(const float* dots, const int* order, float* dweights, int tokens, int k, int slices, void* stream) {
  const int st = experts::checked(tokens, k, slices, TMPI_F32, "expert_dots");
  if (st || !tokens) return st;
  return experts::finish(launch_overlapped(experts::dots_kernel, experts::grid_rows(tokens * k, 8), experts::THREADS, 0, (cudaStream_t)stream, dots, order, dweights,
                                           tokens * k, tokens, k, slices), "expert_dots");
}

}  // extern "C"
