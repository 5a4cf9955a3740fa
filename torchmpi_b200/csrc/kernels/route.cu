// Routing of tokens to experts: the choice of k experts by a token's logits, its weights, the order of all choices by expert, and the
// weights' gradient.
//
// G lanes take a token; a lane holds the logits of experts lane, lane + G, ... as integers that compare like the values, and the best of them apart, so that a
// round of the choice is a maximum over G lanes, a vote for its owner (of equals, which are rare, the lowest index by a second minimum) and a new best of
// the lane that lost its own.  The order by expert is a counting sort in two launches: the first counts the choices of a block of tokens per expert; the second adds the counts of
// the blocks in front, and each warp ranks a contiguous part of the block's choices, 32 at a time, equal ones by their lane, and places them when all ranks are known.  So entries of an expert
// keep their order, and no atomic decides about a place.  Up to SMALL choices one block does both.
//
// Both are bound by latency, chains of dependent shuffles and a few dependent passes over little data, hence the many warps; the choice by instructions too: about 780 for
// four tokens of 64 experts, 8 each, which for 65536 are 13 us at full issue, of 29 measured (the places 18 - 20, the gradient 10).  65536 tokens of 64
// experts, 8 each, forward: 200 us with 8 warps a block, a warp to a token and a thread per expert that walked all choices of its block; 50 with 32
// warps and a warp to a token; 45 with eight lanes to a token, and the gradient 10 where it took 20.  The owner by a vote, where index and value
// were exchanged together, and ranks formed once in place of twice: 8192 tokens of 256 experts 42 -> 36, of 128 21 -> 20, the 65536 of 64 by 1 %.
#include "pdl.cuh"
#include "vec.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>

namespace tmpi {
namespace route {

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int GRADIENT_THREADS = 256;
constexpr int MAX_EXPERTS = 256, MAX_K = 32;
constexpr int MAX_BLOCKS = 148;
constexpr int SMALL = 512;                 // choices that one block counts and places
constexpr uint32_t KEY_NONE = 0x007fffffu; // the key of -inf

struct Problem {
  const void* logits;
  long long ld;                            // elements between rows of the logits
  int tokens, experts, k, renormalize;
  int per_block;                           // tokens of a block
  float* weights;                          // [tokens, k]
  int* chosen;                             // [tokens, k], -1: none
  int* order;                              // [tokens * k], behind the last entry -1
  int* place;                              // [tokens, k], -1: none
  int* offsets;                            // [experts + 1]
  int* counts;                             // [blocks, experts]
};

// Larger values have larger keys; -0 is 0 and NaN is -inf.  0 is no key of a value.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x != x ? __uint_as_float(0xff800000u) : x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int d = G / 2; d; d /= 2) x += __shfl_xor_sync(~0u, x, d);
  return x;
}
template <int G>
__device__ __forceinline__ bool group_any(bool x) {
  const unsigned all = __ballot_sync(~0u, x);
  return G == 32 ? all != 0 : (all >> ((threadIdx.x & 31) & ~(G - 1)) & ((1u << (G & 31)) - 1)) != 0;
}

// One token by G lanes, of which this is lane g with the logits of experts g + G r: chosen and weights of the choices g + G q.  All lanes of the warp;
// `in`: the group has a token.
template <typename T, int G, int R>
__device__ __forceinline__ void choose(const Problem& p, const T* logits, long long token, bool in, int g, int (&chosen)[MAX_K / G], float (&weight)[MAX_K / G]) {
  constexpr int Q = MAX_K / G;
  uint32_t key[R];
  bool nan = false;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = g + G * r;
    const float l = in && e < p.experts ? (float)to_acc<T>(logits[token * p.ld + e]) : 0.f;
    nan |= l != l;
    key[r] = in && e < p.experts ? key_of(l) : 0u;
  }
  nan = group_any<G>(nan);
  uint32_t best = 0;
  int at = g;
  auto renew = [&] {                                               // the lane's best, the lowest index of equals
    best = key[0];
    at = g;
#pragma unroll
    for (int r = 1; r < R; ++r)
      if (key[r] > best) { best = key[r]; at = g + G * r; }
  };
  renew();
  uint32_t top_key = best;
#pragma unroll
  for (int d = G / 2; d; d /= 2) top_key = max(top_key, __shfl_xor_sync(~0u, top_key, d));
  const bool any = top_key > KEY_NONE;
  const float top = of_key(any ? top_key : KEY_NONE + 1);
  float sum = 0.f;
  if (!p.renormalize) {                                            // over all experts
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (any && g + G * r < p.experts) sum += expf(of_key(key[r]) - top);
  }
  constexpr unsigned ALL = G == 32 ? ~0u : (1u << (G & 31)) - 1;
  const int base = (int)(threadIdx.x & 31) & ~(G - 1);             // the group's first lane
  float mine[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    chosen[q] = -1;
    mine[q] = 0.f;
#pragma unroll 1
    for (int j = 0; j < G && q * G + j < p.k; ++j) {
      uint32_t m = best;
#pragma unroll
      for (int d = G / 2; d; d /= 2) m = max(m, __shfl_xor_sync(~0u, m, d));
      const bool there = m > KEY_NONE;                             // else nothing is left that may be used
      const unsigned have = __ballot_sync(~0u, there && best == m) >> base & ALL;
      int i = __shfl_sync(~0u, at, base + __ffs(have) - 1);        // none: any lane's
      if (__any_sync(~0u, (have & (have - 1)) != 0)) {             // equal ones: the lowest index
        i = best == m ? at : p.experts;
#pragma unroll
        for (int d = G / 2; d; d /= 2) i = min(i, __shfl_xor_sync(~0u, i, d));
      }
      if (!there) i = -1;
      if (g == j) {
        chosen[q] = i;
        mine[q] = __uint_as_float(m);
      }
      if (i == at) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (i == g + G * r) key[r] = 0;
        renew();
      }
    }
    mine[q] = chosen[q] >= 0 ? expf(of_key(__float_as_uint(mine[q])) - top) : 0.f;
    if (p.renormalize) sum += mine[q];
  }
  sum = group_sum<G>(sum);
#pragma unroll
  for (int q = 0; q < Q; ++q) weight[q] = nan ? __uint_as_float(0x7fffffffu) : chosen[q] >= 0 ? mine[q] / sum : 0.f;
}

// The tokens of this block: choices and weights to memory, counts per expert to shared memory (cleared by the caller).
template <typename T, int G, int R>
__device__ __forceinline__ void choose_block(const Problem& p, const T* logits, int* counts) {
  const int g = threadIdx.x % G, group = threadIdx.x / G;
  const long long t0 = (long long)blockIdx.x * p.per_block, t1 = min((long long)p.tokens, t0 + p.per_block);
  for (long long tw = t0 + (group & ~(32 / G - 1)); tw < t1; tw += THREADS / G) {      // the same for a warp
    const long long t = tw + (group & (32 / G - 1));
    const bool in = t < t1;
    int c[MAX_K / G];
    float w[MAX_K / G];
    choose<T, G, R>(p, logits, t, in, g, c, w);
#pragma unroll
    for (int q = 0; q < MAX_K / G; ++q)
      if (in && g + G * q < p.k) {
        p.chosen[t * p.k + g + G * q] = c[q];
        p.weights[t * p.k + g + G * q] = w[q];
        if (c[q] >= 0) atomicAdd(&counts[c[q]], 1);                // a count: the order of the additions does not matter
      }
  }
}

// The lanes whose choice is the same, by one vote for each bit of an expert's number (a warp-wide match goes through the different values one by one:
// 65536 tokens of 64 experts, 8 each, took 18.8 us to place out of a cold cache, 14.6 so).  c < 0: no choice, nothing that counts.
__device__ __forceinline__ unsigned same_choice(int c, int bits) {
  unsigned same = __ballot_sync(~0u, c >= 0);
  for (int b = 0; b < bits; ++b) {
    const unsigned set = __ballot_sync(~0u, c >> b & 1);
    same &= c >> b & 1 ? set : ~set;
  }
  return same;
}

struct Place {
  int base[WARPS][MAX_EXPERTS + 1];        // a warp's choices of an expert, then the place of the next of them; padded, for a warp reads a column
  int start[MAX_EXPERTS];                  // the place of the block's first choice of an expert
  int warp_sums[WARPS];
};

// f(choice, whether there is one, its index in the list) for each of this warp's part of the block's choices, 32 at a time
template <typename F>
__device__ __forceinline__ void for_choices(const Problem& p, F f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long e0 = (long long)blockIdx.x * p.per_block * p.k, e1 = min((long long)p.tokens * p.k, e0 + (long long)p.per_block * p.k);
  const long long part = ((long long)p.per_block * p.k + WARPS - 1) / WARPS, w0 = e0 + warp * part, w1 = min(e1, w0 + part);
  constexpr int U = 4;                     // loads in flight
  for (long long i0 = w0; i0 < w1; i0 += 32 * U) {
    int c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = i0 + 32 * u + lane < w1 ? p.chosen[i0 + 32 * u + lane] : -2;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + 32 * u >= w1) break;
      f(c[u], i0 + 32 * u + lane);
    }
  }
}

// Places of this block's choices.  All threads; `s.base` is cleared here.  counts [blocks, experts] (or the block's own), of `blocks` blocks.
__device__ __forceinline__ void place_block(const Problem& p, Place& s, const int* counts, int blocks) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = lane; e < p.experts; e += 32) s.base[warp][e] = 0;
  // an expert's choices in all blocks and in those in front: up to 32 threads share an expert
  int share = 32;
  while (share * p.experts > THREADS) share /= 2;
  const int expert = tid / share;
  int before = 0, total = 0;
  if (expert < p.experts) {
#pragma unroll 8
    for (int b = tid % share; b < blocks; b += share) {
      const int c = counts[(long long)b * p.experts + expert];
      if (b < (int)blockIdx.x) before += c;
      total += c;
    }
  }
  for (int d = 1; d < share; d *= 2) {
    before += __shfl_xor_sync(~0u, before, d);
    total += __shfl_xor_sync(~0u, total, d);
  }
  const bool first = tid % share == 0;
  int sum = first ? total : 0;                                     // inclusive prefix over the experts
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int v = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += v;
  }
  if (lane == 31) s.warp_sums[warp] = sum;
  __syncthreads();                                                 // and base is clear
  int front = s.warp_sums[lane];                                   // every warp scans the warps' sums
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int v = __shfl_up_sync(~0u, front, d);
    if (lane >= d) front += v;
  }
  const int used = __shfl_sync(~0u, front, 31);
  front = __shfl_sync(~0u, front, (warp + 31) & 31);
  const int begin = (warp ? front : 0) + sum - total;              // in the first thread of an expert
  if (first && expert < p.experts) {
    s.start[expert] = begin + before;
    if (blockIdx.x == 0) {
      p.offsets[expert] = begin;
      if (expert == p.experts - 1) p.offsets[p.experts] = used;
    }
  }
  int* mine = s.base[warp];
  const int bits = 32 - __clz(p.experts - 1);                      // none for one expert
  for_choices(p, [&](int c, long long entry) {                     // a choice's rank among those of this warp; kept where its place will be
    const unsigned same = same_choice(c, bits);
    int rank = -1;
    if (c >= 0) rank = mine[c] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (c >= 0 && lane == __ffs(same) - 1) mine[c] += __popc(same);
    __syncwarp();
    if (c >= -1) p.place[entry] = rank;
  });
  __syncthreads();
  for (int e = warp; e < p.experts; e += WARPS) {                  // a warp to an expert: the counts of the block's warps, each behind those in front
    const int n = s.base[lane][e];
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += v;
    }
    s.base[lane][e] = s.start[e] + upto - n;
  }
  __syncthreads();
  for_choices(p, [&](int c, long long entry) {                     // the same thread has the same choices
    if (c < 0) return;
    const int at = mine[c] + p.place[entry];
    p.order[at] = (int)entry;
    p.place[entry] = at;
  });
  for (long long i = used + (long long)blockIdx.x * THREADS + tid; i < (long long)p.tokens * p.k; i += (long long)gridDim.x * THREADS) p.order[i] = -1;
}

template <typename T, int G, int R>
__global__ void __launch_bounds__(THREADS) choose_kernel(const Problem p) {
  __shared__ int counts[MAX_EXPERTS];
  const T* logits = (const T*)p.logits;
  wait_previous(logits);
  for (int e = threadIdx.x; e < p.experts; e += THREADS) counts[e] = 0;
  __syncthreads();
  choose_block<T, G, R>(p, logits, counts);
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += THREADS) p.counts[(long long)blockIdx.x * p.experts + e] = counts[e];
}

__global__ void __launch_bounds__(THREADS) place_kernel(const Problem p) {
  __shared__ Place s;
  const int* counts = p.counts;
  wait_previous(counts);
  place_block(p, s, counts, (int)gridDim.x);
}

template <typename T, int G, int R>
__global__ void __launch_bounds__(THREADS) small_kernel(const Problem p) {
  __shared__ Place s;
  __shared__ int counts[MAX_EXPERTS];
  const T* logits = (const T*)p.logits;
  wait_previous(logits);
  if (threadIdx.x < MAX_EXPERTS) counts[threadIdx.x] = 0;
  __syncthreads();
  choose_block<T, G, R>(p, logits, counts);
  __syncthreads();                                                 // the choices, which this block has written, are read again
  place_block(p, s, counts, 1);
}

// dl of one token by G lanes: of the chosen, w_j (dw_j - sum w dw); with weights over all experts, the others get -p_e sum w dw.
template <typename T, int G, int R>
__global__ void __launch_bounds__(GRADIENT_THREADS) gradient_kernel(const Problem p, const float* dweights, T* dlogits) {
  const T* logits = (const T*)p.logits;
  wait_previous(logits, dweights);
  constexpr int Q = MAX_K / G, PER = GRADIENT_THREADS / G;
  const int g = threadIdx.x % G, group = threadIdx.x / G;
  for (long long tw = (long long)blockIdx.x * PER + (group & ~(32 / G - 1)); tw < p.tokens; tw += (long long)gridDim.x * PER) {      // the same for a warp
    const long long t = tw + (group & (32 / G - 1));
    const bool in = t < p.tokens;
    int c[Q];
    float w[Q], wd[Q], inner = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      c[q] = -1;
      w[q] = wd[q] = 0.f;
      if (in && g + G * q < p.k) {
        c[q] = p.chosen[t * p.k + g + G * q];
        w[q] = p.weights[t * p.k + g + G * q];                     // NaN in a row with a NaN among its logits, whether used or not
        if (c[q] >= 0) wd[q] = w[q] * dweights[t * p.k + g + G * q];
      }
      inner += wd[q];
    }
    float d[R];
#pragma unroll
    for (int r = 0; r < R; ++r) d[r] = 0.f;
    if (!p.renormalize) {
      bool nan = false;
      float top = __uint_as_float(0xff800000u), sum = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        d[r] = in && g + G * r < p.experts ? (float)to_acc<T>(logits[t * p.ld + g + G * r]) : __uint_as_float(0xff800000u);
        nan |= d[r] != d[r];
        top = fmaxf(top, d[r]);
      }
#pragma unroll
      for (int k = G / 2; k; k /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, k));
      nan = group_any<G>(nan);
      const bool any = top > __uint_as_float(0xff800000u);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        d[r] = any ? expf(d[r] - top) : 0.f;
        sum += d[r];
      }
      sum = group_sum<G>(sum);
      inner = group_sum<G>(inner);
      const float scale = nan ? __uint_as_float(0x7fffffffu) : any ? -inner / sum : 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) d[r] = nan ? scale : d[r] * scale;
    } else {
      inner = group_sum<G>(inner);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (in && g + G * r < p.experts) dlogits[t * p.experts + g + G * r] = from_acc<T>((typename AccOf<T>::type)d[r]);
    __syncwarp();                                                  // the chosen ones' are written over it: their p is their weight either way
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (c[q] >= 0) dlogits[t * p.experts + c[q]] = from_acc<T>((typename AccOf<T>::type)(wd[q] - w[q] * inner));
  }
}

static int blocks_of(int tokens, int k) {
  if ((long long)tokens * k <= SMALL) return 1;
  return (int)std::min<long long>(MAX_BLOCKS, ((long long)tokens + 31) / 32);
}

template <int G_, int R_> struct Form { static constexpr int G = G_, R = R_; };
// f(lanes to a token and logits to a lane)
template <typename F>
static cudaError_t by_experts(int experts, F f) {
  if (experts <= 8) return f(Form<8, 1>());
  if (experts <= 16) return f(Form<8, 2>());
  if (experts <= 32) return f(Form<8, 4>());
  if (experts <= 64) return f(Form<8, 8>());
  if (experts <= 128) return f(Form<16, 8>());
  return f(Form<32, 8>());
}

template <typename T>
static cudaError_t forward_t(Problem p, cudaStream_t s) {
  const int blocks = blocks_of(p.tokens, p.k);
  p.per_block = (p.tokens + blocks - 1) / blocks;
  return by_experts(p.experts, [&](auto n) {
    using N = decltype(n);
    if (blocks == 1) return launch_overlapped(small_kernel<T, N::G, N::R>, 1, THREADS, 0, s, p);
    const cudaError_t e = launch_overlapped(choose_kernel<T, N::G, N::R>, blocks, THREADS, 0, s, p);
    return e == cudaSuccess ? launch_overlapped(place_kernel, blocks, THREADS, 0, s, p) : e;
  });
}

template <typename T>
static cudaError_t gradient_t(const Problem& p, const float* dweights, void* dlogits, cudaStream_t s) {
  return by_experts(p.experts, [&](auto n) {
    using N = decltype(n);
    constexpr int per = GRADIENT_THREADS / N::G;
    const int blocks = (int)std::min<long long>(148 * 8, ((long long)p.tokens + per - 1) / per);
    return launch_overlapped(gradient_kernel<T, N::G, N::R>, blocks, GRADIENT_THREADS, 0, s, p, dweights, (T*)dlogits);
  });
}

static int checked(int tokens, int experts, int k, int64_t ld, const char* what) {
  if (tokens < 0 || experts < 1 || k < 1 || k > experts || ld < experts) return fail(TMPI_ERR_INVALID, "%s: %d of %d experts for %d tokens", what, k, experts, tokens);
  if (experts > MAX_EXPERTS || k > MAX_K) return fail(TMPI_ERR_UNSUPPORTED, "%s: at most %d experts, %d for a token", what, MAX_EXPERTS, MAX_K);
  if ((long long)tokens * k > 1LL << 30) return fail(TMPI_ERR_UNSUPPORTED, "%s: %d tokens of %d experts", what, tokens, k);
  return TMPI_OK;
}

}  // namespace route
}  // namespace tmpi

using namespace tmpi;

extern "C" {

int tmpi_route_limits(int* experts, int* k) {
  *experts = route::MAX_EXPERTS;
  *k = route::MAX_K;
  return TMPI_OK;
}

// ints of workspace
size_t tmpi_route_workspace_bytes(int tokens, int experts, int k) {
  const int blocks = route::blocks_of(tokens, k);
  return blocks > 1 ? sizeof(int) * (size_t)blocks * experts : 0;
}

// logits [tokens, experts] of `dtype`, rows ld elements apart -> weights, chosen, place [tokens, k], order [tokens * k], offsets [experts + 1]
int tmpi_route(const void* logits, int64_t ld, int tokens, int experts, int k, int renormalize, int dtype, float* weights, int* chosen, int* order,
               int* place, int* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = route::checked(tokens, experts, k, ld, "route");
  if (st) return st;
  if (workspace_bytes < tmpi_route_workspace_bytes(tokens, experts, k)) return fail(TMPI_ERR_INVALID, "route: workspace too small");
  route::Problem p{};
  p.logits = logits; p.ld = ld; p.tokens = tokens; p.experts = experts; p.k = k; p.renormalize = renormalize;
  p.weights = weights; p.chosen = chosen; p.order = order; p.place = place; p.offsets = offsets; p.counts = (int*)workspace;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  switch (dtype) {
    case TMPI_BF16: e = route::forward_t<__nv_bfloat16>(p, s); break;
    case TMPI_F16: e = route::forward_t<__half>(p, s); break;
    case TMPI_F32: e = route::forward_t<float>(p, s); break;
    default: return fail(TMPI_ERR_UNSUPPORTED, "route: dtype %d", dtype);
  }
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "route launch: %s", cudaGetErrorString(e));
}

// dlogits [tokens, experts] of `dtype`, dense, from dweights [tokens, k] and what the forward gave
int tmpi_route_gradient(const void* logits, int64_t ld, int tokens, int experts, int k, int renormalize, int dtype, const float* weights, const int* chosen,
                        const float* dweights, void* dlogits, void* stream) {
  const int st = route::checked(tokens, experts, k, ld, "route_gradient");
  if (st || !tokens) return st;
  route::Problem p{};
  p.logits = logits; p.ld = ld; p.tokens = tokens; p.experts = experts; p.k = k; p.renormalize = renormalize;
  p.weights = const_cast<float*>(weights); p.chosen = const_cast<int*>(chosen);
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  switch (dtype) {
    case TMPI_BF16: e = route::gradient_t<__nv_bfloat16>(p, dweights, dlogits, s); break;
    case TMPI_F16: e = route::gradient_t<__half>(p, dweights, dlogits, s); break;
    case TMPI_F32: e = route::gradient_t<float>(p, dweights, dlogits, s); break;
    default: return fail(TMPI_ERR_UNSUPPORTED, "route_gradient: dtype %d", dtype);
  }
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "route_gradient launch: %s", cudaGetErrorString(e));
}

}  // extern "C"
