// Products of matrices in 8 bits with a scale for each block of 128 (fp8.cuh) on CTA pairs: C[M,N] = act(A[M,K] B[N,K]^T + bias), sums in fp32.
//
// tcgen05.mma with block scales multiplies e4m3 numbers and, for each row and 32 elements of K, by the two operands' powers of two, which it
// reads from tensor memory: sums of all blocks stay in one accumulator, and the loop is that of the bf16 product (gemm_pair.cuh) at half
// the bytes and twice the rate.  Two CTAs of a cluster share a tile of 256 x 256 (or 256 x 128): each stages 128 rows of A and half of B's, 32 KB for
// 128 of K, and one thread of the even CTA issues for both.
//
// The scales come as 512 bytes for 128 rows and four blocks of K, with the stage of the first of the four.  tcgen05.cp spreads them into four
// columns of each CTA's tensor memory (its own rows of A, all columns' rows of B), behind the MMAs that were issued before and ahead of those that follow;
// two sets are used in turn.  The instruction descriptor says which of the four bytes of a column is meant.
//
// Tensor memory: two accumulators of 256 columns would take all of it.  They overlap by 64: the first has columns 0 to 255, the second 192 to
// 447, the scales lie from 448 on.  An epilogue reads the shared columns first and says so (`shared_free`), and the next tile's MMAs
// wait for that alone, not for the whole accumulator.
//
// Measured (us, bf16 results): 8192^3 366 - 380, 2.9 - 3.0 PFLOP/s, bound by the MMAs and the power limit; 8192 x 4096 x 1024 plain 31 - 33 (its MMAs alone
// 21: of each tile 1.25 us are not hidden, for a cause that is not known; the epilogue's warps wait for the accumulator for half of their time), with the GELU 39 - 40, with the
// pre-activation beside it 46 - 47: bound by the epilogue.  fp16 33, 42, 48; fp32 47, 45, 61, twice the bytes to store.
//
// Few tiles leave SMs idle: K is then cut into slices whose fp32 sums a second kernel adds, in order, and rounds (bit-reproducible).
#include "fp8.cuh"
#include "gelu.cuh"
#include "pdl.cuh"
#include "sm100_ptx.cuh"
#include "vec.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>
#include <mutex>
#include <type_traits>

namespace tmpi {

int make_tmap_box(CUtensorMap* map, int bytes, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows, uint32_t box_cols);
int make_tmap_words(CUtensorMap* map, const void* base, uint64_t rows);
int gemm_sm_count();
int* gemm_status_word();

namespace gemm8 {

constexpr int BM = 128, BN = 256, BK = 128, UMMA_K = 32;
constexpr int A_BYTES = BM * BK, B_BYTES = BN / 2 * BK, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int SF_BYTES = fp8::TILE_BYTES, SF_STAGE = 3 * SF_BYTES;          // 128 rows of A, up to 256 of B
constexpr int COLS = 32;                                                    // of a slice of the epilogue
constexpr int TMEM_COLS = 512, SHARED_COLS = 64, ACC1 = BN - SHARED_COLS, SF_COL = ACC1 + BN, SF_SET = 12;
constexpr int FIRST = SHARED_COLS / COLS;                                   // slices in the columns that the accumulators share
constexpr unsigned long long kWaitBudgetNs = 4000000000ull;

enum { PLAIN = 0, WITH_GELU = 1, GELU_AND_Z = 2 };

template <typename T, int MODE> struct Layout {
  static constexpr int OUTPUTS = MODE == GELU_AND_Z ? 2 : 1;
  static constexpr int GROUPS = sizeof(T) == 4 && MODE == GELU_AND_Z ? 2 : 4;      // of four epilogue warps
  static constexpr int THREADS = 64 + GROUPS * 128;
  static constexpr int TILE = 32 * COLS * sizeof(T);                               // staging of a warp and output
  static constexpr size_t STAGING = (size_t)OUTPUTS * GROUPS * 4 * TILE;
  static constexpr int STAGES = STAGING > 32768 ? 4 : 5;
  static constexpr size_t SF_AT = (size_t)STAGES * STAGE_BYTES, STAGING_AT = (SF_AT + (size_t)STAGES * SF_STAGE + 1023) / 1024 * 1024;
  static constexpr size_t SHARED_AT = STAGING_AT + STAGING;
  static constexpr size_t BYTES = SHARED_AT + 256 + 1024;
  static_assert(BYTES <= 232448, "shared memory of one CTA");
};

struct Shared {
  uint64_t full[5], empty[5], acc_full[2], acc_empty[2], shared_free[2];
  uint32_t tmem_base;
  int error;
};
static_assert(sizeof(Shared) <= 256, "the barriers' place");

struct Problem {
  int M, N, k_blocks;
  int tiles_m, tiles_n;        // of 256 rows, of bn columns
  int bn;                      // columns of a tile: 256, 192 or 128
  int slices, slice_blocks;    // K blocks of a slice, a multiple of four
  int slice_rows;              // rows between the slices' results
  int by_tma;                  // the results' rows are 16-byte multiples
  const void* bias;
  void *c, *z;
  const float* sums;           // [sum_tiles, M]: their sums over the first go to db, of the type db_type, while the first K blocks are under way; or null
  void* db;
  int sum_tiles, db_type;
  int* status;
};

__device__ __forceinline__ void give_up(Shared* sh, const Problem& p, int where) {
  atomicExch(&sh->error, where);
  if (p.status) atomicCAS(p.status, 0, 1100 + where);
}

// Eight rows of tiles at a time, so that the clusters running together share panels of B in L2; all tiles of a slice before the next slice.
struct Item { int m_tile, n_tile, slice; };
__device__ __forceinline__ bool item_of(const Problem& p, int t, Item* it) {
  const int tiles = p.tiles_m * p.tiles_n;
  if (t >= tiles * p.slices) return false;
  it->slice = t / tiles;
  t -= it->slice * tiles;
  constexpr int BAND = 8;
  const int band = t / (BAND * p.tiles_n), rows = min(BAND, p.tiles_m - band * BAND), r = t - band * BAND * p.tiles_n;
  it->m_tile = band * BAND + r % rows;
  it->n_tile = r / rows;
  return true;
}

// D[tmem] (+)= A B^T scaled by the powers of two in tensor memory, e4m3, fp32 sums, both CTAs; one thread issues.
__device__ __forceinline__ void mma_scaled_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// 32 rows of 16 bytes from shared memory into four columns of all lanes (each 32 lanes the same), in both CTAs
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// descriptor of 8-row groups of 16 bytes, 128 bytes apart, without a swizzle
__device__ __forceinline__ uint64_t scales_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// e4m3 x e4m3, both K-major, scales of type e8m0; the numbers of the scales' bytes are added per instruction (bits 29 and 4)
__device__ __forceinline__ uint32_t instruction(int M, int N) { return (uint32_t)(N >> 3) << 17 | 1u << 23 | (uint32_t)(M >> 4) << 24; }

template <int STAGES>
__device__ __forceinline__ void producer(Shared* sh, unsigned char* tiles, unsigned char* sf, const Problem& p, const CUtensorMap* ma, const CUtensorMap* mb, const CUtensorMap* msa,
                                         const CUtensorMap* msb, uint32_t rank, int cluster, int clusters) {
  const int groups = (p.k_blocks + fp8::GROUP - 1) / fp8::GROUP, half = p.bn / 2, b_tiles = (p.bn + 127) / 128;      // 192 columns from a multiple of 64 on: two
  const uint32_t tx = 2 * (A_BYTES + half * BK), tx_scales = 2 * (1 + b_tiles) * SF_BYTES;
  int stage = 0;
  uint32_t phase = 0;
  Item it;
  for (int t = cluster; item_of(p, t, &it); t += clusters) {
    const int a_row = (it.m_tile * 2 + (int)rank) * BM, b_row = it.n_tile * p.bn + (int)rank * half;
    const int kb1 = min(p.k_blocks, (it.slice + 1) * p.slice_blocks);
    for (int kb = it.slice * p.slice_blocks; kb < kb1; ++kb) {
      if (!sm100::mbar_wait(&sh->empty[stage], phase ^ 1, kWaitBudgetNs, &sh->error)) { give_up(sh, p, 1); return; }
      unsigned char* dst = tiles + (size_t)stage * STAGE_BYTES;
      const uint32_t full0 = sm100::map_to_cta(&sh->full[stage], 0);
      const bool scales = (kb & (fp8::GROUP - 1)) == 0;
      if (rank == 0) sm100::mbar_expect_tx(&sh->full[stage], tx + (scales ? tx_scales : 0));          // both CTAs' bytes
      sm100::tma_load_2d_pair(dst, ma, kb * BK, a_row, full0);
      sm100::tma_load_2d_pair(dst + A_BYTES, mb, kb * BK, b_row, full0);
      if (scales) {              // rows of tiles that do not exist read as zero
        unsigned char* s = sf + (size_t)stage * SF_STAGE;
        const int g = kb / fp8::GROUP;
        sm100::tma_load_2d_pair(s, msa, 0, (it.m_tile * 2 + (int)rank) * groups + g, full0);
        for (int j = 0; j < b_tiles; ++j) sm100::tma_load_2d_pair(s + (1 + j) * SF_BYTES, msb, 0, (it.n_tile * p.bn / 128 + j) * groups + g, full0);
      }
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
  }
}

// One thread of the even CTA.
template <int STAGES>
__device__ __forceinline__ void issuer(Shared* sh, unsigned char* tiles, unsigned char* sf, const Problem& p, int cluster, int clusters) {
  const uint32_t idesc = instruction(2 * BM, p.bn);
  const bool overlap = p.bn == BN;
  int stage = 0, set = 0, n = 0;
  uint32_t phase = 0;
  Item it;
  for (int t = cluster; item_of(p, t, &it); t += clusters, ++n) {
    const int acc = n & 1;
    if (!sm100::mbar_wait(&sh->acc_empty[acc], ((n >> 1) & 1) ^ 1, kWaitBudgetNs, &sh->error)) { give_up(sh, p, 2); return; }
    if (overlap && n && !sm100::mbar_wait(&sh->shared_free[acc ^ 1], ((n - 1) >> 1) & 1, kWaitBudgetNs, &sh->error)) { give_up(sh, p, 3); return; }
    sm100::tc_fence_after();
    const uint32_t d = sh->tmem_base + (acc ? (overlap ? ACC1 : p.bn) : 0);
    const int kb0 = it.slice * p.slice_blocks, kb1 = min(p.k_blocks, kb0 + p.slice_blocks);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait(&sh->full[stage], phase, kWaitBudgetNs, &sh->error)) { give_up(sh, p, 4); return; }
      sm100::tc_fence_after();
      const int part = kb & (fp8::GROUP - 1);
      if (part == 0) {
        set ^= 1;
        const uint32_t s = sm100::smem_u32(sf + (size_t)stage * SF_STAGE), to = sh->tmem_base + SF_COL + set * SF_SET;
        copy_scales_pair(to, scales_desc(s));
        copy_scales_pair(to + 4, scales_desc(s + SF_BYTES));
        if (p.bn > 128) copy_scales_pair(to + 8, scales_desc(s + 2 * SF_BYTES));
      }
      // 192 columns may start at the third of a tile's four groups of 32 rows
      const uint32_t sfa = sh->tmem_base + SF_COL + set * SF_SET, sfb = sfa + 4 + (it.n_tile * p.bn % 128) / 32, a = sm100::smem_u32(tiles + (size_t)stage * STAGE_BYTES), b = a + A_BYTES;
      const uint32_t desc = idesc | (uint32_t)part << 29 | (uint32_t)part << 4;
#pragma unroll
      for (int k = 0; k < BK / UMMA_K; ++k)
        mma_scaled_pair(d, sm100::make_desc_sw128(a + k * UMMA_K), sm100::make_desc_sw128(b + k * UMMA_K), desc, sfa, sfb, (kb - kb0) | k);
      sm100::umma_commit_pair(sm100::map_to_cta(&sh->empty[stage], 0));
      sm100::umma_commit_pair(sm100::map_to_cta(&sh->empty[stage], 1));
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
    sm100::umma_commit_pair(sm100::map_to_cta(&sh->acc_full[acc], 0));
    sm100::umma_commit_pair(sm100::map_to_cta(&sh->acc_full[acc], 1));
  }
}

template <typename T> __device__ __forceinline__ uint32_t two(float a, float b);
template <> __device__ __forceinline__ uint32_t two<__nv_bfloat16>(float a, float b) { return attn_util::pack_bf16(__float_as_uint(a), __float_as_uint(b)); }
template <> __device__ __forceinline__ uint32_t two<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 untwo(uint32_t w);
template <> __device__ __forceinline__ float2 untwo<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 untwo<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// gelu of two rounded values, in a word of them; bf16 ones are `gelu_arguments`
template <typename T>
__device__ __forceinline__ uint32_t gelu_word(uint32_t w) {
  const float2 f = untwo<T>(w);
  float y0, y1;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) attn_util::unpack2(shared_gelu2(attn_util::pack2(__float_as_uint(f.x), __float_as_uint(f.y))), y0, y1);          // results of 8 bits: the quicker form (gelu.cuh)
  else gelu_value2(f.x, f.y, &y0, &y1);
  return two<T>(y0, y1);
}
// The Phi of that form stops at 2^-60: of what lies below -1024 nothing may be left, and -inf times nothing is no number.  Both are rare: a minimum for each word tells whether a thread has any.
template <int WORDS>
__device__ __forceinline__ void gelu_arguments(uint32_t (&w)[WORDS]) {
  uint32_t least = w[0];
#pragma unroll
  for (int j = 1; j < WORDS; ++j) asm("min.bf16x2 %0, %0, %1;" : "+r"(least) : "r"(w[j]));
  const float2 f = untwo<__nv_bfloat16>(least);
  if (f.x < -1024.f || f.y < -1024.f) {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) {
      if ((w[j] & 0xffffu) == 0xff80u) w[j] |= 0x7fu;
      if (w[j] >> 16 == 0xff80u) w[j] |= 0x7f0000u;
      asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w[j]) : "r"(0xc480c480u));
    }
  }
}

// Four (two) groups of four warps in each CTA take the tile's slices of 32 columns in turn.  A warp has 32 rows of a slice: it stages them in shared memory and
// stores them through the TMA unit by itself, so that the warps meet nowhere.
template <typename T, int MODE>
__device__ __forceinline__ void epilogue(Shared* sh, unsigned char* staging, const Problem& p, const T* bias, const float* sums, int group, int quarter, int lane, uint32_t rank, int cluster, int clusters,
                                         const CUtensorMap* map_c, const CUtensorMap* map_z) {
  using L = Layout<T, MODE>;
  constexpr int WORDS = COLS * sizeof(T) / 4, ROW = COLS * sizeof(T), PIECES = ROW / 16;
  const bool overlap = p.bn == BN;
  const int parts = p.bn / COLS;
  unsigned char* stg = staging + (size_t)(group * 4 + quarter) * L::OUTPUTS * L::TILE;
  const int swizzle = ROW == 128 ? lane & 7 : (lane >> 1) & 3;
  Item it;
  int n = 0;
  for (int t = cluster; item_of(p, t, &it); t += clusters, ++n) {
    const int acc = n & 1;
    if (MODE == PLAIN && sums && group == 0 && it.n_tile == 0 && it.slice == 0) {
      const int row = (it.m_tile * 2 + (int)rank) * BM + quarter * 32 + lane;
      if (row < p.M) {
        float s = 0.f;
#pragma unroll 8
        for (int i = 0; i < p.sum_tiles; ++i) s += sums[(size_t)i * p.M + row];
        if (p.db_type == TMPI_BF16) ((__nv_bfloat16*)p.db)[row] = __float2bfloat16_rn(s);
        else if (p.db_type == TMPI_F16) ((__half*)p.db)[row] = __float2half_rn(s);
        else ((float*)p.db)[row] = s;
      }
      __syncwarp();
    }
    if (!sm100::mbar_wait_warp(&sh->acc_full[acc], (n >> 1) & 1, kWaitBudgetNs, &sh->error)) { give_up(sh, p, 5); break; }
    sm100::tc_fence_after();
    const int row0 = (it.m_tile * 2 + (int)rank) * BM + quarter * 32, out0 = row0 + it.slice * p.slice_rows;
    const uint32_t t_base = sh->tmem_base + ((uint32_t)(quarter * 32) << 16) + (acc ? (overlap ? ACC1 : p.bn) : 0);
#pragma unroll 1
    for (int i = group; i < parts; i += L::GROUPS) {
      const int c0 = (overlap && !acc ? parts - 1 - i : i) * COLS, col0 = it.n_tile * p.bn + c0;
      const bool inside = col0 < p.N && row0 < p.M;              // the same in all lanes
      uint32_t r[COLS], w[WORDS];
      if (inside) {
        sm100::tmem_ld_32x32(t_base + c0, r);
        sm100::tmem_ld_wait();
      }
      if (overlap && i < FIRST) {       // the columns that the next tile shares have been read
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive_cluster_no_stores(sm100::map_to_cta(&sh->shared_free[acc], 0));
      }
      if (!inside) continue;
      float* v = reinterpret_cast<float*>(r);
      if (bias) {
        if (col0 + COLS <= p.N && ((uintptr_t)bias & 15) == 0) {
#pragma unroll
          for (int j = 0; j < PIECES; ++j) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(bias + col0) + j);
            const uint32_t b[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if constexpr (sizeof(T) == 2) {
                const float2 f = untwo<T>(b[q]);
                v[8 * j + 2 * q] += f.x;
                v[8 * j + 2 * q + 1] += f.y;
              } else {
                v[4 * j + q] += __uint_as_float(b[q]);
              }
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < COLS; ++j)
            if (col0 + j < p.N) v[j] += (float)to_acc<T>(bias[col0 + j]);
        }
      }
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        if constexpr (sizeof(T) == 2) w[j] = two<T>(v[2 * j], v[2 * j + 1]);
        else w[j] = r[j];
      }
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the stores before have read the staging
      __syncwarp();
      auto put = [&](int which) {
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
          *reinterpret_cast<uint4*>(stg + which * L::TILE + lane * ROW + ((u ^ swizzle) << 4)) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
      };
      if (MODE != WITH_GELU) put(0);
      if (MODE != PLAIN) {              // the GELU of what is rounded
        if constexpr (sizeof(T) == 2) {
          if constexpr (std::is_same_v<T, __nv_bfloat16>) gelu_arguments(w);
#pragma unroll
          for (int j = 0; j < WORDS; ++j) w[j] = gelu_word<T>(w[j]);
        } else {
#pragma unroll
          for (int j = 0; j < WORDS; j += 2) {
            float y0, y1;
            gelu_value2(__uint_as_float(w[j]), __uint_as_float(w[j + 1]), &y0, &y1);
            w[j] = __float_as_uint(y0);
            w[j + 1] = __float_as_uint(y1);
          }
        }
        put(MODE == GELU_AND_Z ? 1 : 0);
      }
      if (p.by_tma) {
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          sm100::tma_store_2d(MODE == GELU_AND_Z ? map_z : map_c, stg, col0, out0);
          if (MODE == GELU_AND_Z) sm100::tma_store_2d(map_c, stg + L::TILE, col0, out0);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else {                          // rows that start anywhere: consecutive elements by consecutive lanes
        __syncwarp();
#pragma unroll 1
        for (int o = 0; o < L::OUTPUTS; ++o) {
          T* out = (T*)(L::OUTPUTS == 2 && o == 0 ? p.z : p.c) + col0 + lane;
          if (col0 + lane < p.N)
            for (int j = 0; j < 32 && row0 + j < p.M; ++j) {
              const int at = lane * (int)sizeof(T), sw = ROW == 128 ? j & 7 : (j >> 1) & 3;
              out[(long long)(row0 + j) * p.N] = *reinterpret_cast<const T*>(stg + o * L::TILE + j * ROW + (((at >> 4) ^ sw) << 4) + (at & 15));
            }
        }
        __syncwarp();
      }
    }
    sm100::tc_fence_before();
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive_cluster_no_stores(sm100::map_to_cta(&sh->acc_empty[acc], 0));
  }
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // read before the CTA gives its shared memory back
}

template <typename T, int MODE>
__global__ void __launch_bounds__(Layout<T, MODE>::THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
               const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_z, const Problem p) {
  using L = Layout<T, MODE>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);      // the same offset in both CTAs
  Shared* sh = (Shared*)(base + L::SHARED_AT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = sm100::cluster_ctarank();
  if (warp == 0 && sm100::elect_one()) {
    sm100::tma_prefetch_desc(&map_a);
    sm100::tma_prefetch_desc(&map_b);
    for (int s = 0; s < L::STAGES; ++s) { sm100::mbar_init(&sh->full[s], 1); sm100::mbar_init(&sh->empty[s], 1); }
    for (int a = 0; a < 2; ++a) {
      sm100::mbar_init(&sh->acc_full[a], 1);
      sm100::mbar_init(&sh->acc_empty[a], 2 * 4 * L::GROUPS);
      sm100::mbar_init(&sh->shared_free[a], 2 * 4 * FIRST);
    }
    sh->error = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc_pair(&sh->tmem_base, TMEM_COLS);
    sm100::tmem_relinquish_pair();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();
  sm100::tc_fence_after();
  const T* bias = (const T*)p.bias;
  const float* sums = p.sums;
  wait_previous(bias, sums);
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  if (warp == 0) {
    if (sm100::elect_one()) producer<L::STAGES>(sh, base, base + L::SF_AT, p, &map_a, &map_b, &map_sa, &map_sb, rank, cluster, clusters);
  } else if (warp == 1) {
    if (rank == 0 && sm100::elect_one()) issuer<L::STAGES>(sh, base, base + L::SF_AT, p, cluster, clusters);
  } else {
    epilogue<T, MODE>(sh, base + L::STAGING_AT, p, bias, sums, (warp - 2) >> 2, warp & 3, lane, rank, cluster, clusters, &map_c, &map_z);
  }
  __syncwarp();
  sm100::tc_fence_before();
  __syncthreads();
  if (sh->error && warp == 0 && sm100::elect_one()) {
    const unsigned long long t0 = sm100::now_ns();
    while (sm100::now_ns() - t0 < 200000000ull) { __nanosleep(1000); }   // copies in flight complete within microseconds
  }
  __syncthreads();
  sm100::cluster_sync();                // neither CTA frees its tensor memory or exits while the other may still signal its barriers
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc_pair(sh->tmem_base, TMEM_COLS);
  }
}

// C = the slices' sums, added in order, with the epilogue of the product.  `ld`: of the sums, a multiple of four.
template <typename T>
__global__ void __launch_bounds__(256) add_slices_kernel(const float* __restrict__ sums, const int slices, const long long slice_elements, const int ld, const T* __restrict__ bias,
                                                         T* __restrict__ c, T* __restrict__ z, const int M, const int N, const int gelu, const bool vec) {
  wait_previous(sums, bias);
  const int per_row = ld / 4;
  const long long items = (long long)M * per_row;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < items; i += (long long)gridDim.x * 256) {
    const int row = (int)(i / per_row), col = (int)(i - (long long)row * per_row) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < slices; ++s) {
      const float4 f = __ldcs(reinterpret_cast<const float4*>(sums + s * slice_elements + (long long)row * ld + col));
      v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
    }
    Pack<T, 4> out, kept;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (bias && col + k < N) v[k] += (float)to_acc<T>(bias[col + k]);
      out.v[k] = kept.v[k] = from_acc<T>((typename AccOf<T>::type)v[k]);
    }
    if (gelu) {
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        float y0, y1;
        gelu_value2((float)to_acc<T>(kept.v[k]), (float)to_acc<T>(kept.v[k + 1]), &y0, &y1);
        out.v[k] = from_acc<T>((typename AccOf<T>::type)y0);
        out.v[k + 1] = from_acc<T>((typename AccOf<T>::type)y1);
      }
    }
    const long long at = (long long)row * N + col;
    if (vec && col + 4 <= N) {
      st_pack<T, 4>(c + at, out);
      if (z) st_pack<T, 4>(z + at, kept);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (col + k < N) {
          c[at + k] = out.v[k];
          if (z) z[at + k] = kept.v[k];
        }
    }
  }
}

// ---------------------------------------------------------------- host side
struct Plan { int bn, slices, slice_blocks, tiles_m, tiles_n; };

static int max_clusters() { return gemm_sm_count() / 2; }

// Columns of a tile, and slices of K, by the time that they take, in us: 3 for the launch and its first loads, and for each round of tiles that for a block of 128 of K
// and that for what the next tile's MMAs do not hide of the epilogue.  Measured: 256 columns 0.371 and 1.25, 192 0.285 and 1.0, 128 0.222 and 1.05 (8192 x 4096 x 1024 in
// 33.1, 36.0, 42.6 us; 8192 x 1024 x 4096 29.3, 33.5, 35.6; 4096 x 1024 x 8192, one round of 64 tiles of 256, 28.0, 39.9, 36.5).  Slices cost a launch and their
// sums' way to memory and back (1024 x 1024 x 8192: 17.4 in four slices, 20.0 in tiles of 128 without).
static Plan plan_of(int M, int N, int k_blocks) {
  struct Width { int columns; double block, tile; };
  constexpr Width widths[] = {{256, 0.371, 1.25}, {192, 0.285, 1.0}, {128, 0.222, 1.05}};
  const int clusters = max_clusters(), tm = (M + 2 * BM - 1) / (2 * BM);
  Plan best{};
  double least = 1e30;
  for (const Width& w : widths) {
    const int tn = (N + w.columns - 1) / w.columns;
    for (int s = 1; s <= 16 && 4 * (s - 1) < k_blocks; ++s) {
      const int per = ((k_blocks + s - 1) / s + 3) / 4 * 4, slices = (k_blocks + per - 1) / per;
      if (slices != s) continue;
      const long long rounds = ((long long)tm * tn * s + clusters - 1) / clusters;
      double us = 3. + rounds * (std::min(per, k_blocks) * w.block + w.tile);
      if (s > 1) us += 2.5 + (double)M * N * 4. * (s + 1) / 4.5e6;
      if (us < least) {
        least = us;
        best = {w.columns, s, per, tm, tn};
      }
    }
  }
  return best;
}

template <typename T, int MODE>
static cudaError_t launch(const CUtensorMap* m, const Problem& p, cudaStream_t stream) {
  static std::once_flag once;
  std::call_once(once, [] { cudaFuncSetAttribute(product_kernel<T, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Layout<T, MODE>::BYTES); });
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  const long long items = (long long)p.tiles_m * p.tiles_n * p.slices;
  cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(items, max_clusters()));
  cfg.blockDim = dim3(Layout<T, MODE>::THREADS);
  cfg.dynamicSmemBytes = Layout<T, MODE>::BYTES; cfg.stream = stream; cfg.attrs = at; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, product_kernel<T, MODE>, m[0], m[1], m[2], m[3], m[4], m[5], p);
}

static int ld_of(int N) { return (N + 3) / 4 * 4; }
static int64_t slice_rows(const Plan& pl) { return (int64_t)pl.tiles_m * 2 * BM; }
static bool too_large(int64_t M, int64_t N, int64_t K) {
  return M < 1 || N < 1 || K < 1 || M > 1 << 30 || N > 1 << 30 || K > 1 << 30 || (double)((M + 255) / 256) * (double)((N + 127) / 128) * 16 > 2e9;
}

template <typename T>
static int run(const void* qa, const void* sa, const void* qb, const void* sb, const void* bias, void* c, void* z, int M, int N, int K, int gelu, void* ws, size_t ws_bytes,
               cudaStream_t stream, const float* sums = nullptr, int sum_tiles = 0, void* db = nullptr, int db_type = 0) {
  const Plan pl = plan_of(M, N, fp8::blocks_of(K));
  const int groups = fp8::groups_of(K), es = sizeof(T);
  Problem p{};
  p.M = M; p.N = N; p.k_blocks = fp8::blocks_of(K);
  p.tiles_m = pl.tiles_m; p.tiles_n = pl.tiles_n; p.bn = pl.bn; p.slices = pl.slices; p.slice_blocks = pl.slice_blocks;
  p.bias = bias; p.c = c; p.z = z;
  p.sums = sums; p.sum_tiles = sum_tiles; p.db = db; p.db_type = db_type;
  p.status = gemm_status_word();
  CUtensorMap m[6];
  int st;
  if ((st = make_tmap_box(&m[0], 1, qa, (uint64_t)M, (uint64_t)fp8::pitch_of(K), BM, BK))) return st;
  if ((st = make_tmap_box(&m[1], 1, qb, (uint64_t)N, (uint64_t)fp8::pitch_of(K), pl.bn / 2, BK))) return st;
  if ((st = make_tmap_words(&m[2], sa, (uint64_t)((M + 127) / 128) * groups))) return st;
  if ((st = make_tmap_words(&m[3], sb, (uint64_t)((N + 127) / 128) * groups))) return st;
  cudaError_t e;
  if (pl.slices > 1) {
    const int ld = ld_of(N);
    if (!ws || ws_bytes < (size_t)pl.slices * slice_rows(pl) * ld * 4) return fail(TMPI_ERR_INVALID, "fp8_product: a workspace of %zu bytes is too small", ws_bytes);
    if ((int64_t)pl.slices * slice_rows(pl) > 0x7fffffff) return fail(TMPI_ERR_UNSUPPORTED, "fp8_product: %d x %d is too large", M, N);
    if ((st = make_tmap_box(&m[4], 4, ws, (uint64_t)pl.slices * slice_rows(pl), (uint64_t)ld, 32, gemm8::COLS))) return st;
    m[5] = m[4];
    p.slice_rows = (int)slice_rows(pl);
    p.by_tma = 1;
    p.bias = nullptr;
    if ((e = launch<float, PLAIN>(m, p, stream)) == cudaSuccess) {
      const long long items = (long long)M * (ld / 4);
      const bool vec = (size_t)N * es % (4 * es) == 0 && !((uintptr_t)c & (4 * es - 1)) && !((uintptr_t)z & (4 * es - 1));
      e = launch_overlapped(add_slices_kernel<T>, (unsigned)std::min<long long>((items + 255) / 256, 148 * 8), 256, 0, stream, (const float*)ws, pl.slices,
                            (long long)slice_rows(pl) * ld, ld, (const T*)bias, (T*)c, (T*)z, M, N, gelu, vec);
    }
  } else {
    p.by_tma = (size_t)N * es % 16 == 0 && all_aligned16({c, z});
    m[4] = m[5] = m[0];                 // not used without by_tma
    if (p.by_tma && (st = make_tmap_box(&m[4], es, c, (uint64_t)M, (uint64_t)N, 32, gemm8::COLS))) return st;
    if (p.by_tma && z && (st = make_tmap_box(&m[5], es, z, (uint64_t)M, (uint64_t)N, 32, gemm8::COLS))) return st;
    e = z ? launch<T, GELU_AND_Z>(m, p, stream) : gelu ? launch<T, WITH_GELU>(m, p, stream) : launch<T, PLAIN>(m, p, stream);
  }
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "fp8_product launch: %s", cudaGetErrorString(e));
}

}  // namespace gemm8
}  // namespace tmpi

using namespace tmpi;

extern "C" {

int tmpi_fp8_product_form(int M, int N, int K, int* columns, int* slices) {
  if (gemm8::too_large(M, N, K)) return fail(TMPI_ERR_INVALID, "fp8_product_form: %d x %d x %d", M, N, K);
  const gemm8::Plan pl = gemm8::plan_of(M, N, fp8::blocks_of(K));
  *columns = pl.bn;
  *slices = pl.slices;
  return TMPI_OK;
}

size_t tmpi_fp8_product_workspace_bytes(int M, int N, int K) {
  if (gemm8::too_large(M, N, K)) return 0;
  const gemm8::Plan pl = gemm8::plan_of(M, N, fp8::blocks_of(K));
  return pl.slices > 1 ? (size_t)pl.slices * gemm8::slice_rows(pl) * gemm8::ld_of(N) * 4 : 0;
}

// c [M, N] of `dtype` = a b^T (+ bias), a [M, K] and b [N, K] in 8 bits (tmpi_fp8_quantize); gelu: the GELU of the rounded sums, which go to z where it is given.
int tmpi_fp8_product(const void* qa, const void* sa, const void* qb, const void* sb, const void* bias, void* c, void* z, int M, int N, int K, int gelu, int dtype, void* ws, size_t ws_bytes,
                     void* stream) {
  if (gemm8::too_large(M, N, K)) return fail(TMPI_ERR_INVALID, "fp8_product: %d x %d x %d", M, N, K);
  if (!all_aligned16({qa, sa, qb, sb, ws})) return fail(TMPI_ERR_INVALID, "fp8_product: operands must be 16-byte aligned");
  if (z && !gelu) return fail(TMPI_ERR_INVALID, "fp8_product: the pre-activation is kept with the GELU");
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case TMPI_BF16: return gemm8::run<__nv_bfloat16>(qa, sa, qb, sb, bias, c, z, M, N, K, gelu, ws, ws_bytes, s);
    case TMPI_F16: return gemm8::run<__half>(qa, sa, qb, sb, bias, c, z, M, N, K, gelu, ws, ws_bytes, s);
    case TMPI_F32: return gemm8::run<float>(qa, sa, qb, sb, bias, c, z, M, N, K, gelu, ws, ws_bytes, s);
  }
  return fail(TMPI_ERR_UNSUPPORTED, "fp8_product: dtype %d", dtype);
}

int tmpi_fp8_product_sums(const void* qa, const void* sa, const void* qb, const void* sb, void* c, const float* sums, int tiles, void* db, int M, int N, int K, int dtype, void* ws,
                          size_t ws_bytes, void* stream) {
  if (gemm8::too_large(M, N, K) || !sums || !db || tiles < 1) return fail(TMPI_ERR_INVALID, "fp8_product_sums: %d x %d x %d, %d rows of sums", M, N, K, tiles);
  if (!all_aligned16({qa, sa, qb, sb, ws})) return fail(TMPI_ERR_INVALID, "fp8_product_sums: operands must be 16-byte aligned");
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case TMPI_BF16: return gemm8::run<__nv_bfloat16>(qa, sa, qb, sb, nullptr, c, nullptr, M, N, K, 0, ws, ws_bytes, s, sums, tiles, db, dtype);
    case TMPI_F16: return gemm8::run<__half>(qa, sa, qb, sb, nullptr, c, nullptr, M, N, K, 0, ws, ws_bytes, s, sums, tiles, db, dtype);
    case TMPI_F32: return gemm8::run<float>(qa, sa, qb, sb, nullptr, c, nullptr, M, N, K, 0, ws, ws_bytes, s, sums, tiles, db, dtype);
  }
  return fail(TMPI_ERR_UNSUPPORTED, "fp8_product_sums: dtype %d", dtype);
}

}  // extern "C"
