// AdamW over many tensors at once, with states in 32 or in 8 bits, and the norm of many gradients.
//
//   g = coefficient * gradient;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   w = (1 - lr decay) w - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// All of it in fp32, w being the fp32 master where there is one (its rounding is then stored as the weight).  t counts a tensor's steps and lies on the
// device, like the clipping coefficient: a captured step can be replayed.
//
// The states of all tensors lie in one buffer each, a tensor's from a multiple of 128 elements on; the tensors' own addresses and extents come as a
// table among the kernel's parameters (32 bytes a tensor), so that a step is one launch without a copy to the device.  Tensors are cut into chunks of 2048 elements,
// a thread eight of them; a block takes chunk after chunk, as many apart as there are blocks, finds the first one's tensor by bisection and forms a
// tensor's rates when it comes to it.  Bound by memory: 354 M elements of bf16 with masters take 1640 us in 32 bits (28 bytes an element, 6.0 TB/s, 0.92 of the copy rate), 1010 in 8
// (16.1, 5.6), where half of the issue slots are taken too; without masters 1230 and 890.
//
// In 8 bits, 128 elements share the largest magnitude among them (fp32), and an element is kept as the root of its share of that, in multiples of 1/127 with
// its sign for m, and of 1/255 for the root of v: m = +-c^2 top / 127^2, sqrt(v) = c^2 top / 255^2.  The root spends the codes evenly over ratios: the
// largest are kept within 0.4 % (m: 0.8 %), what is 1/100 of it within 4 % (8 %), and the least number that is not zero is 1/65025 (1/16129) of it.  Of v it is the root
// that divides the update, and an element whose root is not zero never becomes zero: m / sqrt(v) stays bounded, by a divisor that is then too
// large, not too small.  The scale of a block is not rounded: where all of its averages shrink alike, as without gradients, the codes stay and
// the scale follows (with a scale rounded to a power of two an average would stand still, its step of 1 % being less than half a code).
// A block with an element that is not finite becomes NaN.
#include "attn_util.cuh"
#include "pdl.cuh"
#include "vec.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>
#include <vector>

namespace tmpi {
namespace adamw {

constexpr int THREADS = 256, BLOCK = 128;
constexpr int CHUNK = THREADS * 8;

struct Entry {
  void* param;
  const void* grad;
  uint32_t chunk;        // the first of its chunks
  uint32_t n;            // elements
  uint32_t place;        // of its states, in blocks of 128
  uint32_t which;        // the number of its step count, << 8 | its group | PART | COUNTED
};
static_assert(sizeof(Entry) == 32, "the table's size");
constexpr uint32_t PART = 0x80000000u;        // a further part of a tensor, whose first part counts the step
constexpr uint32_t COUNTED = 0x40000000u;     // that part was in a launch before this one
constexpr int MAX_STEPS = 1 << 22;            // step counts that an entry can name
struct Group { float decay, lr, beta1, beta2, rest1, rest2, log_beta1, log_beta2, eps; const float* device_lr; };      // rest: 1 - beta
constexpr int MAX_GROUPS = 8;

// SMALL fits the 4 KB of parameters that cost least to launch with
constexpr int SMALL = 100, LARGE = 980;
template <int CAP> struct Table {
  Group group[MAX_GROUPS];
  Entry entry[CAP];
};

struct States {
  void *m, *v;                   // fp32, or codes
  float *m_top, *v_top;          // of 8 bits
  float* master;
  int* steps;
  const float* coefficient;      // of the gradients, on the device, or null
  unsigned* counter;             // zero between launches
  float scale;                   // of the gradients
  int entries;
};

// sqrt to within two units in the last place, of subnormals too; `quick_root` takes those for zero
__device__ __forceinline__ float root(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float quick_root(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the entry that a chunk belongs to
template <int CAP>
__device__ __forceinline__ int entry_of(const Table<CAP>& t, int entries, uint32_t chunk) {
  int lo = 0, hi = entries - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.entry[mid].chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// PER consecutive elements, in pieces of 16 bytes at most
template <typename T, int PER>
__device__ __forceinline__ void load(const T* __restrict__ p, int n, bool vec, float* x) {
  if (vec && n >= PER) {
    constexpr int V = PER * sizeof(T) <= 16 ? PER : 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < PER / V; ++j) {
      const Pack<T, V> a = ld_pack<T, V>(p + j * V);
#pragma unroll
      for (int k = 0; k < V; ++k) x[j * V + k] = (float)to_acc<T>(a.v[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = k < n ? (float)to_acc<T>(p[k]) : 0.f;
  }
}
template <typename T, int PER>
__device__ __forceinline__ void store(T* __restrict__ p, int n, bool vec, const float* x) {
  if (vec && n >= PER) {
    constexpr int V = PER * sizeof(T) <= 16 ? PER : 16 / sizeof(T);
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

// a byte as a float through the mantissa of 2^23, and back: rounded to the nearest integer, of which the low byte counts
__device__ __forceinline__ float of_byte(uint32_t w, int k) { return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540u + k)); }
__device__ __forceinline__ uint32_t bytes(const float* r) {
  const uint32_t lo = __byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040), hi = __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
constexpr float LEAST = 7.888609052210118e-31f;          // 2^-100: what a share is divided by at least
constexpr float LEAST_EPS = 1e-37f;                      // an element without any gradient is 0 / (0 + eps): stays, also with eps = 0
constexpr float LEAST_EPS8 = 1e-18f;                     // of 8-bit states, which know no root below 1e-19
constexpr float LEAST_DIVISOR = 2e-38f;                  // the least eps over a large rate: a subnormal divisor counts as zero in `rcp`, and 0 / 0 is no number

// the largest magnitude of 128 elements, of which 128 / PER lanes have PER each; NaN if one is not finite
template <int PER>
__device__ __forceinline__ float block_top(const float (&x)[PER]) {
  float a = attn_util::max_nan(fabsf(x[0]), fabsf(x[1]));
#pragma unroll
  for (int k = 2; k < PER; k += 2) a = attn_util::max3_nan(a, fabsf(x[k]), fabsf(x[k + 1]));
#pragma unroll
  for (int d = 1; d < BLOCK / PER; d *= 2) a = attn_util::max_nan(a, __shfl_xor_sync(~0u, a, d));
  return a < __uint_as_float(0x7f800000u) ? a : __uint_as_float(0x7fffffffu);
}

// four codes of the first moment, and of the second's root
__device__ __forceinline__ void decode_m(uint32_t w, float unit, float* m) {
  w ^= 0x80808080u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float c = of_byte(w, k) - 8388736.f;
    m[k] = c * fabsf(c) * unit;
  }
}
__device__ __forceinline__ void decode_v(uint32_t w, float unit, float* v) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float c = of_byte(w, k) - 8388608.f, r = c * c * unit;
    v[k] = r * r;
  }
}

template <typename T, int BITS, bool MASTER, int CAP>
__global__ void __launch_bounds__(THREADS, 5) step_kernel(const __grid_constant__ Table<CAP> table, const States s, const uint32_t chunks) {
  constexpr int PER = CHUNK / THREADS;
  // Elements of a thread that lie beside each other; its next ones are APART further.  Four, where most bytes are those of fp32, so that a warp's accesses are whole
  // lines (two 16-byte stores beside each other are half sectors for each of the warp's instructions); else all, whose 16-bit loads are then 16 bytes.
  constexpr int RUN = BITS == 32 && (MASTER || sizeof(T) == 4) ? 4 : PER;
  constexpr uint32_t APART = RUN * THREADS;
  __shared__ unsigned ticket;
  wait_previous();
  const float coefficient = s.scale * (s.coefficient ? *s.coefficient : 1.f);
  int at = entry_of(table, s.entries, blockIdx.x);
  // Rates of a group's tensors with the same step count, which most have: formed anew where that changes (for each tensor they took 4 % of a step).
  float seen = -1.f, unbias = 0.f, eps = 0.f, keep = 0.f, b1 = 0.f, b2 = 0.f, a1 = 0.f, a2 = 0.f, unit_m = 0.f, unit_v = 0.f;
  uint32_t seen_group = ~0u;
  for (uint32_t c = blockIdx.x; c < chunks; at = entry_of(table, s.entries, c)) {      // one tensor after another
    const Entry& e = table.entry[at];
    const float t = (float)(s.steps[(e.which & (COUNTED - 1)) >> 8] + (e.which & COUNTED ? 0 : 1));
    const uint32_t e0 = e.chunk, end = at + 1 < s.entries ? table.entry[at + 1].chunk : chunks, extent = e.n, whole = (extent + BLOCK - 1) / BLOCK * BLOCK;
    T* const param = (T*)e.param;
    const T* const grads = (const T*)e.grad;
    const bool vec = (((uintptr_t)param | (uintptr_t)grads) & 15) == 0;
    const size_t place = (size_t)e.place * BLOCK;
    for (; c < end; c += gridDim.x) {
      const uint32_t first = (c - e0) * CHUNK + threadIdx.x * RUN;             // of the tensor
      float grad[PER], w[PER], m[PER], v[PER];
      auto left = [&](int j) { const uint32_t f = first + j * APART; return f < extent ? (int)min((uint32_t)RUN, extent - f) : 0; };
      auto padded = [&](int j) { return first + j * APART < whole ? RUN : 0; };      // the states go on, as zeros, to the end of a block
#pragma unroll
      for (int j = 0; j < PER / RUN; ++j) {
        const size_t p = place + first + j * APART;
        load<T, RUN>(grads + first + j * APART, left(j), vec, grad + RUN * j);
        if (MASTER) load<float, RUN>(s.master + p, padded(j), true, w + RUN * j);
        else load<T, RUN>(param + first + j * APART, left(j), vec, w + RUN * j);
        if constexpr (BITS == 32) {
          load<float, RUN>((const float*)s.m + p, padded(j), true, m + RUN * j);
          load<float, RUN>((const float*)s.v + p, padded(j), true, v + RUN * j);
        }
      }
      const size_t p0 = place + first;
      uint2 cm = make_uint2(0u, 0u), cv = cm;
      float um = 0.f, uv = 0.f;
      if (BITS == 8 && padded(0)) {
        cm = *reinterpret_cast<const uint2*>((const uint8_t*)s.m + p0);
        cv = *reinterpret_cast<const uint2*>((const uint8_t*)s.v + p0);
        um = s.m_top[p0 / BLOCK];
        uv = s.v_top[p0 / BLOCK];
      }
      // behind the loads: a small step is as long as its chain of latencies
      if (t != seen || (e.which & 0xff) != seen_group) {
        seen = t;
        seen_group = e.which & 0xff;
        const Group& g = table.group[seen_group];
        const float lr = g.device_lr ? *g.device_lr : g.lr;
        // The update is m / (sqrt(v) unbias + eps) with the rate lr / (1 - b1^t) in the divisor (a rate below 1e-30, whose inverse may be no number, counts as 0: an
        // infinite divisor), and of what is squared on its way into v the root is taken here.
        const float step = lr / -expm1f(t * g.log_beta1);
        const bool moves = step >= 1e-30f;
        unbias = moves ? rsqrtf(-expm1f(t * g.log_beta2)) / step : 0.f;
        eps = moves ? fmaxf(fmaxf(g.eps, BITS == 8 ? LEAST_EPS8 : LEAST_EPS) / step, LEAST_DIVISOR) : __uint_as_float(0x7f800000u);
        keep = 1.f - lr * g.decay;
        b1 = g.beta1, b2 = g.beta2, a1 = g.rest1 * coefficient, a2 = sqrtf(g.rest2) * coefficient;
        unit_m = b1 * (1.f / 16129.f), unit_v = sqrtf(b2) * (1.f / 65025.f);
      }
      if constexpr (BITS == 8) {                       // times the decay of the averages, which enters the units
        decode_m(cm.x, um * unit_m, m), decode_m(cm.y, um * unit_m, m + 4);
        decode_v(cv.x, uv * unit_v, v), decode_v(cv.y, uv * unit_v, v + 4);
      }
      float r[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const float x = grad[k] * a2;
        m[k] = fmaf(a1, grad[k], BITS == 8 ? m[k] : b1 * m[k]);
        v[k] = fmaf(x, x, BITS == 8 ? v[k] : b2 * v[k]);
        r[k] = BITS == 8 ? quick_root(v[k]) : root(v[k]);
        w[k] = fmaf(-m[k], attn_util::rcp(fmaf(r[k], unbias, eps)), keep * w[k]);
      }
#pragma unroll
      for (int j = 0; j < PER / RUN; ++j) {
        const size_t p = place + first + j * APART;
        store<T, RUN>(param + first + j * APART, left(j), vec, w + RUN * j);
        if (padded(j)) {
          if (MASTER) store<float, RUN>(s.master + p, RUN, true, w + RUN * j);
          if constexpr (BITS == 32) {
            store<float, RUN>((float*)s.m + p, RUN, true, m + RUN * j);
            store<float, RUN>((float*)s.v + p, RUN, true, v + RUN * j);
          }
        }
      }
      if constexpr (BITS == 8) {
        const float mt = block_top<PER>(m), vt = block_top<PER>(r), sm = 16129.f * attn_util::rcp(fmaxf(mt, LEAST)), sv = 65025.f * attn_util::rcp(fmaxf(vt, LEAST));
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          m[k] = copysignf(quick_root(fabsf(m[k]) * sm), m[k]) + 12582912.f;
          r[k] = quick_root(fmaxf(r[k] * sv, __saturatef(r[k] * 3e38f))) + 8388608.f;      // at least 1 for what is not zero
        }
        if (padded(0)) {
          *reinterpret_cast<uint2*>((uint8_t*)s.m + p0) = make_uint2(bytes(m), bytes(m + 4));
          *reinterpret_cast<uint2*>((uint8_t*)s.v + p0) = make_uint2(bytes(r), bytes(r + 4));
          if ((threadIdx.x & (BLOCK / PER - 1)) == 0) {
            s.m_top[p0 / BLOCK] = mt;
            s.v_top[p0 / BLOCK] = vt;
          }
        }
      }
    }
  }
  // The last block to come counts the step.  All others have read the counts then, and need no fence for it: what they read has decided about their branches.
  __syncthreads();
  if (threadIdx.x == 0) ticket = atomicAdd(s.counter, 1u);
  __syncthreads();
  if (ticket == gridDim.x - 1) {
    for (int i = threadIdx.x; i < s.entries; i += THREADS)
      if (!(table.entry[i].which & PART)) s.steps[table.entry[i].which >> 8] += 1;
    if (threadIdx.x == 0) *s.counter = 0;
  }
}

// ---------------------------------------------------------------- the norm of many tensors
// Sums of squares: a thread's in fp32 (a few thousand of them), all others in fp64, in a fixed order.  Bound by memory: 354 M elements in 387 bf16 tensors 152 us, in 20 109
// (0.99 of the copy rate), in fp32 205 and 188 (1.06 and 1.15: the copy writes too).
constexpr int NORM_BLOCKS = 148 * 4;
__host__ __device__ constexpr uint32_t unit_chunks(int element_bytes) { return 32768 / (CHUNK * element_bytes); }

// Eight loads of 16 bytes, 4096 apart, that the compiler does not take apart (it waits for the first before it sends the last otherwise).
__device__ __forceinline__ void load_eight(const void* p, uint32_t (&u)[32]) {
  asm volatile(
      "ld.global.v4.u32 {%0, %1, %2, %3}, [%32];\n\tld.global.v4.u32 {%4, %5, %6, %7}, [%32+4096];\n\t"
      "ld.global.v4.u32 {%8, %9, %10, %11}, [%32+8192];\n\tld.global.v4.u32 {%12, %13, %14, %15}, [%32+12288];\n\t"
      "ld.global.v4.u32 {%16, %17, %18, %19}, [%32+16384];\n\tld.global.v4.u32 {%20, %21, %22, %23}, [%32+20480];\n\t"
      "ld.global.v4.u32 {%24, %25, %26, %27}, [%32+24576];\n\tld.global.v4.u32 {%28, %29, %30, %31}, [%32+28672];"
      : "=&r"(u[0]), "=&r"(u[1]), "=&r"(u[2]), "=&r"(u[3]), "=&r"(u[4]), "=&r"(u[5]), "=&r"(u[6]), "=&r"(u[7]), "=&r"(u[8]), "=&r"(u[9]), "=&r"(u[10]), "=&r"(u[11]), "=&r"(u[12]),
        "=&r"(u[13]), "=&r"(u[14]), "=&r"(u[15]), "=&r"(u[16]), "=&r"(u[17]), "=&r"(u[18]), "=&r"(u[19]), "=&r"(u[20]), "=&r"(u[21]), "=&r"(u[22]), "=&r"(u[23]), "=&r"(u[24]),
        "=&r"(u[25]), "=&r"(u[26]), "=&r"(u[27]), "=&r"(u[28]), "=&r"(u[29]), "=&r"(u[30]), "=&r"(u[31])
      : "l"(p));
}

// What becomes of the sums: norm = scale sqrt(their sum), coefficient = min(1, most / (norm + 1e-6)), NaN staying.
struct Finish {
  float *norm, *coefficient;     // coefficient may be null
  unsigned* counter;             // zero between launches
  float scale, most;
};
// of the first n sums, by all threads of a block
__device__ __forceinline__ void finish_norm(const double* sums, int n, const Finish& f) {
  double d = 0.;
  for (int i = threadIdx.x; i < n; i += THREADS) d += __ldcg(sums + i);
  __shared__ double part[THREADS / 32];
#pragma unroll
  for (int i = 16; i; i >>= 1) d += __shfl_xor_sync(~0u, d, i);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) d += part[i];
    const float r = (float)(fabs((double)f.scale) * sqrt(d));
    *f.norm = r;
    if (f.coefficient) *f.coefficient = f.most / (r + 1e-6f) > 1.f ? 1.f : f.most / (r + 1e-6f);
  }
}

// A block takes units of 32 KB (a few chunks in a row), as many apart as there are blocks, so that many small tensors are shared among all.  Of a unit that is
// not whole, or of several tensors, four chunks at a time are under way (7 M fp32 elements of 67 tensors, with what is made of the sums: 14.3 -> 10.6 us).  Its sum goes to sums[before + block]; with a counter the last block to come takes those of all launches for the norm.
template <typename T, int CAP>
__global__ void __launch_bounds__(THREADS, 4) squares_kernel(const __grid_constant__ Table<CAP> table, const int entries, const uint32_t chunks, double* __restrict__ sums, const int before,
                                                             const Finish finish) {
  constexpr int PER = CHUNK / THREADS, AHEAD = 4;
  wait_previous(sums);
  float a[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) a[k] = 0.f;
  for (uint32_t c0 = blockIdx.x * unit_chunks(sizeof(T)); c0 < chunks; c0 += gridDim.x * unit_chunks(sizeof(T))) {
    const uint32_t c1 = min(chunks, c0 + unit_chunks(sizeof(T)));
    int at = entry_of(table, entries, c0);
    const Entry& e = table.entry[at];
    if (c1 - c0 == unit_chunks(sizeof(T)) && (c1 - e.chunk) * (uint64_t)CHUNK <= e.n && ((uintptr_t)e.grad & 15) == 0) {          // whole, and of one tensor
      constexpr int V = 16 / sizeof(T);
      uint32_t x[32];
      load_eight((const T*)e.grad + (size_t)(c0 - e.chunk) * CHUNK + threadIdx.x * V, x);
#pragma unroll
      for (int j = 0; j < 8 * V; ++j) {
        const float f = (float)to_acc<T>(reinterpret_cast<const T*>(x)[j]);
        a[j % PER] = fmaf(f, f, a[j % PER]);
      }
      continue;
    }
    for (uint32_t c = c0; c < c1; c += AHEAD) {
      float x[AHEAD][PER];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        while (at + 1 < entries && table.entry[at + 1].chunk <= c + u) ++at;
        const Entry& e = table.entry[at];
        const T* const grads = (const T*)e.grad;
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
          const uint32_t first = (c + u - e.chunk) * CHUNK + j * THREADS + threadIdx.x * 4;
          load<T, 4>(grads + first, c + u < c1 && first < e.n ? (int)min(4u, e.n - first) : 0, ((uintptr_t)grads & 15) == 0, x[u] + j);
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int k = 0; k < PER; ++k) a[k] = fmaf(x[u][k], x[u][k], a[k]);
    }
  }
  double d = 0.;
#pragma unroll
  for (int k = 0; k < PER; ++k) d += (double)a[k];
  __shared__ double part[THREADS / 32];
  __shared__ bool last;
#pragma unroll
  for (int i = 16; i; i >>= 1) d += __shfl_xor_sync(~0u, d, i);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) d += part[i];
    __stcg(sums + before + blockIdx.x, d);
    __threadfence();
    last = finish.counter && atomicAdd(finish.counter, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (last) {
    finish_norm(sums, before + (int)gridDim.x, finish);
    if (threadIdx.x == 0) *finish.counter = 0;
  }
}

__global__ void __launch_bounds__(THREADS) norm_kernel(const double* __restrict__ sums, const int n, const Finish finish) {
  wait_previous(sums);
  finish_norm(sums, n, finish);
}

// ---------------------------------------------------------------- what 8-bit states stand for
template <typename T>
__global__ void __launch_bounds__(THREADS) values_kernel(const uint8_t* __restrict__ m, const float* __restrict__ m_top, const uint8_t* __restrict__ v, const float* __restrict__ v_top,
                                                         T* __restrict__ mo, T* __restrict__ vo, const long long items) {
  wait_previous(m, m_top, v, v_top);
  const long long i = (long long)blockIdx.x * THREADS + threadIdx.x;
  if (i >= items) return;
  const uint2 cm = reinterpret_cast<const uint2*>(m)[i], cv = reinterpret_cast<const uint2*>(v)[i];
  const float um = m_top[i / 16] * (1.f / 16129.f), uv = v_top[i / 16] * (1.f / 65025.f);
  float a[8], b[8];
  decode_m(cm.x, um, a), decode_m(cm.y, um, a + 4);
  decode_v(cv.x, uv, b), decode_v(cv.y, uv, b + 4);
  store<T, 8>(mo + i * 8, 8, true, a);
  store<T, 8>(vo + i * 8, 8, true, b);
}

// ---------------------------------------------------------------- host side
// Tables for the tensors [i, ...) until one is full; returns the next tensor and how much of it is in the table.
struct Filled { int entries; uint32_t chunks; int finished; };          // finished: tensors whose last element is in the table or before
constexpr int64_t MOST = int64_t(1) << 30;               // elements of an entry

template <int CAP>
static Filled fill(Table<CAP>* t, const tmpi_adamw_tensor_t* tensors, int count, int* i, int64_t* done, bool groups) {
  Filled f{0, 0, 0};
  uint32_t counted = *done ? COUNTED : 0u;
  while (*i < count && f.entries < CAP) {
    const tmpi_adamw_tensor_t& x = tensors[*i];
    if (x.n <= 0) { ++*i; continue; }                    // counted by the caller's steps as soon as it has elements
    const int64_t n = std::min(x.n - *done, MOST);
    if (f.chunks + (uint64_t)(n + CHUNK - 1) / CHUNK > 0x7fffffffull) break;
    const int64_t bytes = *done * x.element_bytes;
    Entry& e = t->entry[f.entries++];
    e.param = x.param ? (char*)x.param + bytes : nullptr;
    e.grad = (const char*)x.grad + bytes;
    e.chunk = f.chunks;
    e.n = (uint32_t)n;
    e.place = (uint32_t)((x.offset + *done) / BLOCK);
    e.which = groups ? (uint32_t)x.step << 8 | (uint32_t)x.group | (*done ? PART : 0u) | counted : 0u;
    f.chunks += (uint32_t)((n + CHUNK - 1) / CHUNK);
    *done += n;
    if (*done >= x.n) { ++*i; ++f.finished; *done = 0; counted = 0u; }
  }
  return f;
}

template <typename T, int CAP>
static cudaError_t launch_step(const Table<CAP>& t, const States& s, int bits, uint32_t chunks, cudaStream_t stream) {
  constexpr bool MASTERS = sizeof(T) == 2;               // fp32 has none
  const bool master = MASTERS && s.master;
  const auto kernel = bits == 8 ? (master ? step_kernel<T, 8, MASTERS, CAP> : step_kernel<T, 8, false, CAP>) : (master ? step_kernel<T, 32, MASTERS, CAP> : step_kernel<T, 32, false, CAP>);
  return launch_overlapped(kernel, std::min<uint32_t>(chunks, 148 * 5), THREADS, 0, stream, t, s, chunks);
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

template <int CAP, typename F>
static cudaError_t each_table(const tmpi_adamw_tensor_t* tensors, int count, const tmpi_adamw_group_t* groups, int ngroups, F f) {
  Table<CAP> t;
  for (int g = 0; g < ngroups; ++g) {
    const tmpi_adamw_group_t& x = groups[g];
    t.group[g] = {x.weight_decay, x.lr, x.beta1, x.beta2, x.rest1, x.rest2, x.log_beta1, x.log_beta2, x.eps, x.device_lr};
  }
  int i = 0;
  int64_t done = 0;
  while (i < count) {
    const Filled filled = fill<CAP>(&t, tensors, count, &i, &done, ngroups > 0);
    if (!filled.entries) continue;
    const cudaError_t e = f(t, filled);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace adamw
}  // namespace tmpi

using namespace tmpi;

extern "C" {

int tmpi_adamw_max_groups(void) { return adamw::MAX_GROUPS; }

int tmpi_adamw_step(const tmpi_adamw_tensor_t* tensors, int count, const tmpi_adamw_group_t* groups, int ngroups, const tmpi_adamw_states_t* states, int bits, int dtype, void* stream) {
  if (count < 0 || ngroups < 1 || ngroups > adamw::MAX_GROUPS || (bits != 8 && bits != 32)) return fail(TMPI_ERR_INVALID, "adamw: %d groups, %d bits", ngroups, bits);
  if (!all_aligned16({states->m, states->v, states->master})) return fail(TMPI_ERR_INVALID, "adamw: states must be 16-byte aligned");
  for (int i = 0; i < count; ++i)
    if (tensors[i].offset % adamw::BLOCK || tensors[i].offset / adamw::BLOCK + (tensors[i].n + 127) / 128 > 0xffffffffLL || tensors[i].group < 0 || tensors[i].group >= ngroups || tensors[i].step < 0 ||
        tensors[i].step >= adamw::MAX_STEPS)
      return fail(TMPI_ERR_INVALID, "adamw: tensor %d has no place among the states", i);
  adamw::States s{states->m, states->v, states->m_top, states->v_top, states->master, states->steps, states->coefficient, states->counter, states->scale, 0};
  return adamw::by_type(dtype, "adamw", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    if (sizeof(T) == 4 && s.master) return cudaErrorInvalidValue;
    auto run = [&](const auto& table, const adamw::Filled& f) {
      s.entries = f.entries;
      return adamw::launch_step<T>(table, s, bits, f.chunks, (cudaStream_t)stream);
    };
    return count <= adamw::SMALL ? adamw::each_table<adamw::SMALL>(tensors, count, groups, ngroups, run) : adamw::each_table<adamw::LARGE>(tensors, count, groups, ngroups, run);
  });
}

// Sums of squares of `count` tensors into sums [tmpi_norm_sums(count)], of which *used were written.  A launch takes SMALL entries at least, and the tensors of a GPU (less than
// 2^38 bytes) have not more than 256 entries beside their first ones.
int tmpi_norm_sums(int count) { return (count / adamw::SMALL + 5) * adamw::NORM_BLOCKS; }
// The norm of `used` sums, and a clipping coefficient where it has a place.  With a counter (a word that is zero between launches, of one stream's launches) the last launch of
// tmpi_norm_squares does that too, of `used` sums before and its own.
int tmpi_norm_squares(const tmpi_adamw_tensor_t* tensors, int count, int dtype, double* sums, int* used, const tmpi_norm_finish_t* finish, void* stream) {
  if (count < 0 || *used < 0) return fail(TMPI_ERR_INVALID, "norm: %d tensors", count);
  int rest = 0;
  for (int i = 0; i < count; ++i) rest += tensors[i].n > 0;
  return adamw::by_type(dtype, "norm", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    auto run = [&](const auto& table, const adamw::Filled& f) {
      constexpr int CAP = sizeof(table.entry) / sizeof(adamw::Entry);
      const uint32_t unit = adamw::unit_chunks(sizeof(T)), blocks = std::min<uint32_t>((f.chunks + unit - 1) / unit, adamw::NORM_BLOCKS);
      adamw::Finish last{};
      rest -= f.finished;
      if (finish && !rest) last = {finish->norm, finish->coefficient, finish->counter, finish->scale, finish->most};
      const cudaError_t e = launch_overlapped(adamw::squares_kernel<T, CAP>, blocks, adamw::THREADS, 0, (cudaStream_t)stream, table, f.entries, f.chunks, sums, *used, last);
      *used += (int)blocks;
      return e;
    };
    return count <= adamw::SMALL ? adamw::each_table<adamw::SMALL>(tensors, count, nullptr, 0, run) : adamw::each_table<adamw::LARGE>(tensors, count, nullptr, 0, run);
  });
}
int tmpi_norm_finish(const double* sums, int n, float scale, float most, float* norm, float* coefficient, void* stream) {
  const cudaError_t e = launch_overlapped(adamw::norm_kernel, 1, adamw::THREADS, 0, (cudaStream_t)stream, sums, n, adamw::Finish{norm, coefficient, nullptr, scale, most});
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "norm launch: %s", cudaGetErrorString(e));
}

// blocks of 128 elements -> m and v in `dtype`
int tmpi_adamw_values(const void* m, const float* m_top, const void* v, const float* v_top, void* mo, void* vo, int64_t blocks, int dtype, void* stream) {
  if (blocks < 0 || blocks > (int64_t)1 << 31) return fail(TMPI_ERR_INVALID, "adamw_values: %lld blocks", (long long)blocks);
  if (!blocks) return TMPI_OK;
  if (!all_aligned16({m, v, mo, vo})) return fail(TMPI_ERR_INVALID, "adamw_values: tensors must be 16-byte aligned");
  return adamw::by_type(dtype, "adamw_values", [&](auto* type) -> cudaError_t {
    using T = std::remove_pointer_t<decltype(type)>;
    const long long items = blocks * (adamw::BLOCK / 8);
    return launch_overlapped(adamw::values_kernel<T>, (unsigned)((items + adamw::THREADS - 1) / adamw::THREADS), adamw::THREADS, 0, (cudaStream_t)stream, (const uint8_t*)m, m_top,
                             (const uint8_t*)v, v_top, (T*)mo, (T*)vo, items);
  });
}

}  // extern "C"
