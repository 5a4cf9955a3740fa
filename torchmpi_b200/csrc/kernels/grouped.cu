// Matrix products grouped by expert, on CTA pairs (gemm_pair.cuh): the rows offsets[e] <= r < offsets[e + 1] of x belong to expert e.
//   y_r = x_r w_e^T + b_e      (w [experts, N, K] as it lies; backward's dx_r = dy_r w_e reads it MN-major)
//   dw_e = sum of dy_r^T x_r,  db_e = sum of dy_r
// The offsets are read on the device: nothing is known of the groups on the host, and no call waits for it.
//
// Rows products.  A group is cut into tiles of 256 rows x bn columns, counted by every CTA for itself (a prefix sum over the experts in shared memory);
// the tiles of all groups form one list, dealt to persistent clusters in turn.  A tile's rows may start anywhere: the row coordinate of a TMA
// load has no alignment rule, and rows beyond the group's end, of other experts, only reach accumulator rows that are not stored.  A CTA
// whose part of the tile has at most 32 rows loads 32, and none without rows, so that few rows cost little beside the weights.  Whole parts are
// stored through TMA tiles, others row by row.  The weight is a 3-D tensor: what a box reads beyond the matrix of its expert is zero, not the next
// expert's, whose infinities would come back as NaN.
//
// The weights' gradient has the rows as its K.  The last 64 rows of a group may hold rows of the next one: a warp of each CTA waits
// for that block's loads and overwrites those rows with zeros in both operands (zero times infinity is not zero), as far as the
// MMAs read; the issuer waits for both CTAs' warps there.  db is
// summed by the epilogue warps under the tile's MMAs, in fp32 and in short chains, as in linear_bwd.cu.  Experts without rows get zeros.
#include "act8.cuh"
#include "attn_util.cuh"
#include "gemm_pair.cuh"
#include "pdl.cuh"
#include "../include/tmpi_c_api.h"
#include "../runtime/common.h"
#include <algorithm>
#include <mutex>

namespace tmpi {

int make_tmap_bf16(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows);
int make_tmap_bf16_3d(CUtensorMap* map, const void* base, uint64_t outer, uint64_t rows, uint64_t cols, uint32_t box_rows, uint32_t box_cols);
int make_tmap_box(CUtensorMap* map, int bytes, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows, uint32_t box_cols);
int gemm_sm_count();
int* gemm_status_word();

namespace grouped {

using namespace gemm2;
constexpr int MAX_EXPERTS = 256;
constexpr int FEW = 32;                                 // rows of the smaller box of x
constexpr int SLICE = 64;                               // columns of a tile that an epilogue warp takes

// PLAIN32: the sum in fp32.  GRADIENT8 / 16: the sum is the gradient of a GELU's value, whose input z was kept in 8 bits or in bf16.
enum { PLAIN = 0, GELU_ONLY = 1, WITH_GELU = 2, KEEP8 = 3, PLAIN32 = 4, GRADIENT8 = 5, GRADIENT16 = 6 };

struct Problem {
  const int* offsets;        // [experts + 1]; null: one expert with all rows
  int rows, experts, K, N;   // of x; N: columns of the result
  int bn, tiles_n, k_blocks;
  int slices, per;           // PLAIN32 with few rows: parts of K, of `per` blocks, each with a result of its own [slices, rows, N]
  const __nv_bfloat16* bias; // [experts, N] or null
  __nv_bfloat16* y;          // [rows, N]; GRADIENT: dz
  float* y32;                // PLAIN32
  void* z;                   // WITH_GELU, GRADIENT16: the pre-activation [rows, N]; KEEP8, GRADIENT8: its e4m3 numbers
  uint8_t* scale;            // and their scales
  __nv_bfloat16* h;          // GRADIENT: weight times gelu(z)
  const float* row_weights;  // GRADIENT: [rows] or null (ones)
  float* dots;               // GRADIENT: sums over 64 (few rows: 32) columns of gradient times gelu(z), where dots_at says; or null
  int wide;                  // every row of y, z, h starts on a 32-byte boundary
  int q_rows16;              // 8 bits: every row of z starts on a 16-byte boundary, as TMA tiles and 16-byte loads need
  int scale_pairs;           // 8 bits: two scales of a row that belong to 64 columns lie in one aligned 16-bit word
  int* status;
};

// Four groups of four epilogue warps: a group takes 64 columns of a tile, a warp of it 32 rows, which it stages and stores by itself.  With two groups,
// whose warps met at barriers around the stores, a GELU epilogue ran at 1.1 instructions per cycle and SM and was longer than its tile's MMAs:
// 16384 x 4096 x 1024 127 us with a GELU, 176 with an 8-bit checkpoint beside it, 103 plain.
constexpr int ROW_GROUPS = 4, ROW_THREADS = 64 + ROW_GROUPS * 128;
// Stages of the operand ring: a warp has a staging buffer of 32 rows x 64 bytes, or two (one of 128 bytes) where it has two results or fp32.
__host__ __device__ constexpr int stages_of(int mode) { return mode == PLAIN || mode == GELU_ONLY ? 6 : 5; }
__host__ __device__ constexpr int staging_of(int mode) { return mode == PLAIN || mode == GELU_ONLY ? 2048 : 4096; }

struct Sh {
  uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
  uint64_t kept[4 * ROW_GROUPS];                        // GRADIENT8: what was kept of z for a warp's part of the tile
  uint32_t tmem_base;
  int error;
  int warp_sums[8];
  int tile_end[MAX_EXPERTS];                            // tiles of the experts up to and with this one
};
constexpr size_t SMEM = (size_t)STAGES * STAGE_BYTES + 32768 + 1024 + 1408;
static_assert(5 * STAGE_BYTES + 16 * 4096 == 6 * STAGE_BYTES + 16 * 2048 && 6 * STAGE_BYTES + 16 * 2048 == STAGES * STAGE_BYTES + 32768, "staging");
static_assert(sizeof(Sh) <= 1408 && SMEM <= 232448, "shared memory of one CTA");

// Offsets as given, but inside the tensor and not before the group's start: wrong ones give wrong results, never an access outside.
struct Group { int r0, r1; };
__device__ __forceinline__ Group group_of(const int* __restrict__ offsets, int rows, int e) {
  if (!offsets) return {0, rows};
  const int r0 = min(max(__ldg(offsets + e), 0), rows);
  return {r0, min(max(__ldg(offsets + e + 1), r0), rows)};
}

struct Unit {
  int e, n_blk;
  int row0, end;             // of the pair's tile: first row, end of the group
  __device__ __forceinline__ int part_rows(uint32_t rank) const { return min(max(end - row0 - (int)rank * BM, 0), BM); }
};

// Four slices of a row lie side by side, [slices / 4, rows, 4]: a warp, with a slice of 32 rows, writes to 16 sectors, and whoever adds a row's slices reads
// 16 bytes of each.
__device__ __forceinline__ long long dots_at(int slice, int rows, long long row) { return ((long long)(slice >> 2) * rows + row) * 4 + (slice & 3); }

template <typename S>
__device__ __forceinline__ void give_up(S* sh, int* status, int where) {
  atomicExch(&sh->error, where);
  if (status) atomicCAS(status, 0, 1000 + where);
}

// Tiles of `rows` rows.  All threads of the CTA; ends with a barrier.
__device__ __forceinline__ void count_tiles(Sh* sh, const Problem& p, const int* offsets, int rows) {
  const int e = threadIdx.x, lane = e & 31, warp = e >> 5;
  int tiles = 0;
  if (e < p.experts) {
    const Group g = group_of(offsets, p.rows, e);
    tiles = (g.r1 - g.r0 + rows - 1) / rows * p.tiles_n;
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int v = __shfl_up_sync(~0u, tiles, d);
    if (lane >= d) tiles += v;
  }
  if (lane == 31 && warp < 8) sh->warp_sums[warp] = tiles;
  __syncthreads();
  if (e < p.experts) {
    for (int w = 0; w < warp; ++w) tiles += sh->warp_sums[w];
    sh->tile_end[e] = tiles;
  }
  __syncthreads();
}

// f(unit, number in this cluster's list) for each tile of this cluster until it returns false
template <typename F>
__device__ __forceinline__ void for_tiles(const Sh* sh, const Problem& p, const int* offsets, F f) {
  const int total = sh->tile_end[p.experts - 1], step = (int)(gridDim.x >> 1);
  int e = 0, it = 0;
  for (int t = (int)(blockIdx.x >> 1); t < total; t += step, ++it) {
    if (sh->tile_end[e] <= t) {                          // the first expert that ends behind t, which is behind e
      int hi = p.experts - 1;
      ++e;
      while (e < hi) {
        const int mid = (e + hi) >> 1;
        if (sh->tile_end[mid] > t) hi = mid;
        else e = mid + 1;
      }
    }
    const int begin = e ? sh->tile_end[e - 1] : 0;
    const Group g = group_of(offsets, p.rows, e);
    Unit u;
    int m_tile;
    band_order(t - begin, (sh->tile_end[e] - begin) / p.tiles_n, p.tiles_n, &m_tile, &u.n_blk);
    u.e = e;
    u.row0 = g.r0 + m_tile * 2 * BM;
    u.end = g.r1;
    if (!f(u, it)) return;
  }
}

// bytes of x that a part with this many rows loads for one K block
__device__ __forceinline__ uint32_t a_bytes(int rows) { return rows > FEW ? A_BYTES : rows > 0 ? FEW * BK * 2 : 0; }

struct Ring { int stage; uint32_t phase; };
template <int N>
__device__ __forceinline__ void advance(Ring* r) { if (++r->stage == N) { r->stage = 0; r->phase ^= 1; } }

// One thread in each CTA.
template <int NST, bool B_MN>
__device__ __forceinline__ void produce(Sh* sh, unsigned char* tiles, const Problem& p, const int* offsets, const CUtensorMap* ma, const CUtensorMap* ma_few,
                                        const CUtensorMap* mb, uint32_t rank) {
  const int half = p.bn / 2;
  const bool two = half > 64;
  const uint32_t b_tx = 2 * (B_MN ? (two ? B_BYTES : B_BYTES / 2) : half * BK * 2);
  Ring ring{0, 0};
  for_tiles(sh, p, offsets, [&](const Unit& u, int) -> bool {
    const int mine = u.part_rows(rank), a_row0 = u.row0 + (int)rank * BM, n0 = u.n_blk * p.bn + (int)rank * half;
    const uint32_t tx = b_tx + a_bytes(u.part_rows(0)) + a_bytes(u.part_rows(1));
    for (int kb = 0; kb < p.k_blocks; ++kb) {
      const int stage = ring.stage;
      if (!sm100::mbar_wait(&sh->empty[stage], ring.phase ^ 1, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 31); return false; }
      unsigned char* dst = tiles + (size_t)stage * STAGE_BYTES;
      const uint32_t full0 = sm100::map_to_cta(&sh->full[stage], 0);
      if (rank == 0) sm100::mbar_expect_tx(&sh->full[stage], tx);              // both CTAs' bytes
      if (mine > 0) sm100::tma_load_2d_pair(dst, mine > FEW ? ma : ma_few, kb * BK, a_row0, full0);
      if (!B_MN) {
        sm100::tma_load_3d_pair(dst + A_BYTES, mb, kb * BK, n0, u.e, full0);
      } else {
        sm100::tma_load_3d_pair(dst + A_BYTES, mb, n0, kb * BK, u.e, full0);
        if (two) sm100::tma_load_3d_pair(dst + A_BYTES + B_BYTES / 2, mb, n0 + 64, kb * BK, u.e, full0);
      }
      advance<NST>(&ring);
    }
    return true;
  });
}

// One thread of the even CTA.
template <int NST, bool B_MN>
__device__ __forceinline__ void issue(Sh* sh, unsigned char* tiles, const Problem& p, const int* offsets) {
  const uint32_t idesc = sm100::make_idesc_f16(2 * BM, p.bn, true, B_MN, false);
  Ring ring{0, 0};
  for_tiles(sh, p, offsets, [&](const Unit&, int it) -> bool {
    const int acc = it & 1;
    if (!sm100::mbar_wait(&sh->acc_empty[acc], ((it >> 1) & 1) ^ 1, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 32); return false; }
    sm100::tc_fence_after();
    const uint32_t d = sh->tmem_base + (uint32_t)acc * BN;
    for (int kb = 0; kb < p.k_blocks; ++kb) {
      const int stage = ring.stage;
      if (!sm100::mbar_wait(&sh->full[stage], ring.phase, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 33); return false; }
      sm100::tc_fence_after();
      const uint32_t a = sm100::smem_u32(tiles + (size_t)stage * STAGE_BYTES), b = a + A_BYTES;
#pragma unroll
      for (int k = 0; k < BK / UMMA_K; ++k) {
        const uint64_t da = sm100::make_desc_sw128(a + k * UMMA_K * 2);
        const uint64_t db = B_MN ? sm100::make_desc_sw128_mn(b + k * UMMA_K * 128, B_BYTES / 2, 1024) : sm100::make_desc_sw128(b + k * UMMA_K * 2);
        sm100::umma_f16_pair(d, da, db, idesc, (uint32_t)kb | (uint32_t)k);
      }
      sm100::umma_commit_pair(sm100::map_to_cta(&sh->empty[stage], 0));
      sm100::umma_commit_pair(sm100::map_to_cta(&sh->empty[stage], 1));
      advance<NST>(&ring);
    }
    sm100::umma_commit_pair(sm100::map_to_cta(&sh->acc_full[acc], 0));
    sm100::umma_commit_pair(sm100::map_to_cta(&sh->acc_full[acc], 1));
    return true;
  });
}

// 32-bit words to consecutive addresses: 32 bytes at once where rows start on such a boundary (a whole sector of L2 per lane), else 16 or 8.
__device__ __forceinline__ void store32(void* to, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// 32 bf16 columns of a row, `left` of them inside it (a multiple of 8)
__device__ __forceinline__ void store_row(__nv_bfloat16* to, const uint32_t (&w)[16], int left, bool wide) {
  if (wide && left >= 32) {
    store32(to, w);
    store32(to + 16, w + 8);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (8 * j < left) reinterpret_cast<uint4*>(to)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  }
}
// 32 e4m3 columns
__device__ __forceinline__ void store_row8(uint8_t* to, const uint32_t (&q)[8], int left, bool wide) {
  if (wide && left >= 32) {
    store32(to, q);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (8 * j < left) reinterpret_cast<uint2*>(to)[j] = make_uint2(q[2 * j], q[2 * j + 1]);
  }
}
// the same read, where rows start on 8-byte boundaries alone (others come through the TMA unit)
__device__ __forceinline__ void load_row8(const uint8_t* from, uint32_t (&q)[8], int left) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint2 v = 8 * j < left ? reinterpret_cast<const uint2*>(from)[j] : make_uint2(0u, 0u);
    q[2 * j] = v.x; q[2 * j + 1] = v.y;
  }
}
__device__ __forceinline__ void pack_row(const float (&v)[32], uint32_t (&w)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = attn_util::pack_bf16(__float_as_uint(v[2 * j]), __float_as_uint(v[2 * j + 1]));
}

// The sixteen epilogue warps of each CTA.  A thread has a row of the tile, and its warp works on 32 of its columns at a time, without a word to
// the others.  A warp whose 32 rows all belong to the group stores through its own staging and the TMA unit, others from registers, row by row.  (Stores of
// registers, 32 bytes a lane, for all of them: the shared memory's data path, which the MMAs read their operands through, moved 16 bytes a cycle for
// them; two results of 8192 x 4096 kept it busy half of the time, and the launch took as much longer.)  The GELU is that of the fp32 sum, and so is the
// 8-bit checkpoint, whose blocks of 32 columns a thread has to itself.
template <int MODE>
__device__ __forceinline__ void finish(Sh* sh, unsigned char* staging, const Problem& p, const int* offsets, const __nv_bfloat16* bias_all, const float* row_weights,
                                       const CUtensorMap* map_y, const CUtensorMap* map_z, const CUtensorMap* map_kept, uint32_t rank, int group, int quarter, int lane) {
  constexpr bool GRADIENT = MODE == GRADIENT8 || MODE == GRADIENT16;
  const int row = quarter * 32 + lane, N = p.N, bn = p.bn, blocks = (N + 31) / 32;
  uint64_t* kept_bar = &sh->kept[group * 4 + quarter];
  uint32_t kept_phase = 0;
  const bool wide = p.wide != 0;
  for_tiles(sh, p, offsets, [&](const Unit& u, int it) -> bool {
    const int acc = it & 1, rows = u.part_rows(rank), c0 = group * SLICE, col0 = u.n_blk * bn + c0;
    const bool busy = rows > quarter * 32 && c0 < bn && col0 < N;                 // of this warp
    const bool mine = busy && row < rows, whole = rows >= quarter * 32 + 32;
    const int warp_row = u.row0 + (int)rank * BM + quarter * 32;
    // staged results: rows of 64 bytes (128 in fp32), 16-byte pieces permuted as the tensor maps' swizzle has it
    auto reuse = [&](int pending) {                      // all but the last `pending` stores have been read out of the staging
      if (lane == 0) {
        if (pending) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      }
      __syncwarp();
    };
    auto stage = [&](int buffer, const uint32_t (&w)[16]) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(staging + buffer * 2048 + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    };
    auto send = [&](const CUtensorMap* map, int buffer, int col) {
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        sm100::tma_store_2d(map, staging + buffer * 2048, col, warp_row);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    };
    const long long row_at = (long long)u.row0 + (int)rank * BM + row;
    const __nv_bfloat16* bias = bias_all ? bias_all + (long long)u.e * N : nullptr;
    // GRADIENT: what was kept of z comes through the TMA unit into the warp's staging while the products are under way, and is in registers before
    // results are staged there.  16384 x 4096 x 1024, each pair measured in turn: 8 bits 136.0 us (139.7 with 16-byte loads, four lanes to a row, handed over
    // through the staging; 147 against 141 with a lane's own row), 16 bits 140.6 (147.0 with a lane's own row).
    float weight = 1.f, dot = 0.f;
    uint32_t kept[MODE == GRADIENT8 ? 16 : GRADIENT ? 32 : 1], scales = 0x0101u;
    const bool by_tma = MODE == GRADIENT16 || (MODE == GRADIENT8 && p.q_rows16);
    if (GRADIENT) {                                      // while the products are under way
      if (by_tma && busy && lane == 0) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        sm100::mbar_expect_tx(kept_bar, MODE == GRADIENT8 ? 2048 : 4096);
        sm100::tma_load_2d(staging, map_kept, col0, warp_row, kept_bar);
        if (MODE == GRADIENT16) sm100::tma_load_2d(staging + 2048, map_kept, col0 + 32, warp_row, kept_bar);
      }
      if (mine) {
        if (row_weights) weight = __ldg(row_weights + row_at);
        if (MODE == GRADIENT8) {
          const uint8_t* at = p.scale + row_at * blocks + col0 / 32;
          if (p.scale_pairs) scales = *reinterpret_cast<const uint16_t*>(at);
          else scales = at[0] | (col0 + 32 < N ? (uint32_t)at[1] << 8 : 0x0100u);
          if (!by_tma) {
#pragma unroll
            for (int h = 0; h < 2; ++h) load_row8((const uint8_t*)p.z + row_at * N + col0 + 32 * h, *reinterpret_cast<uint32_t(*)[8]>(&kept[8 * h]), N - col0 - 32 * h);
          }
        }
      }
    }
    if (!sm100::mbar_wait_warp(&sh->acc_full[acc], (it >> 1) & 1, kWaitBudgetNs, &sh->error)) { give_up(sh, p.status, 34); return false; }
    sm100::tc_fence_after();
    const uint32_t t_base = sh->tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)acc * BN + c0;
    auto release = [&] {                                 // the accumulator has been read
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive_cluster_no_stores(sm100::map_to_cta(&sh->acc_empty[acc], 0));
    };
    if (!busy) { release(); return true; }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int col = col0 + 32 * half, left = N - col;
      if (half && left <= 0) { release(); break; }
      uint32_t r[32];
      if (GRADIENT && by_tma && !half) {
        if (!sm100::mbar_wait_warp(kept_bar, kept_phase, kWaitBudgetNs, &sh->error)) { give_up(sh, p.status, 35); return false; }
        kept_phase ^= 1;
#pragma unroll
        for (int j = 0; j < (MODE == GRADIENT8 ? 4 : 8); ++j) {
          const uint4 v = *reinterpret_cast<const uint4*>(staging + (j >> 2) * 2048 + lane * 64 + (((j & 3) ^ (lane >> 1 & 3)) << 4));
          kept[4 * j] = v.x; kept[4 * j + 1] = v.y; kept[4 * j + 2] = v.z; kept[4 * j + 3] = v.w;
        }
        __syncwarp();
      }
      sm100::tmem_ld_32x32(t_base + 32 * half, r);
      uint4 b[4];
      if (!GRADIENT && bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = __ldg(reinterpret_cast<const uint4*>(bias + (8 * j < left ? col + 8 * j : 0)));      // what lies behind N is never read
      }
      sm100::tmem_ld_wait();
      if (half) release();
      float v[32];
      if (!GRADIENT && bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x[4] = {b[j].x, b[j].y, b[j].z, b[j].w};
#pragma unroll
          for (int q = 0; q < 4; ++q)
            attn_util::unpack2(attn_util::add2(attn_util::pack2(r[8 * j + 2 * q], r[8 * j + 2 * q + 1]), attn_util::pack2(x[q] << 16, x[q] & 0xffff0000u)), v[8 * j + 2 * q],
                               v[8 * j + 2 * q + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
      }
      uint32_t w[16];
      if (MODE == PLAIN32) {
        if (whole) {
          reuse(0);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(staging + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          send(map_y, 0, col);
        } else if (mine) {
          float* to = p.y32 + row_at * N + col;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (8 * j < left) store32(to + 8 * j, reinterpret_cast<const uint32_t*>(v) + 8 * j);
        }
        continue;
      }
      if (MODE == WITH_GELU) {
        pack_row(v, w);
        if (whole) {
          reuse(1);
          stage(1, w);
          send(map_z, 1, col);
        } else if (mine) {
          store_row((__nv_bfloat16*)p.z + row_at * N + col, w, left, wide);
        }
      }
      if ((MODE == KEEP8 || GRADIENT) && left < 32) {    // columns behind N do not count: an infinity times the weight's zeros there is NaN
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j >= left) v[j] = 0.f;
      }
      if (MODE == KEEP8) {
        uint32_t q[8];
        const uint32_t byte = act8::pack_block(v, q);
        scales = half ? scales | byte << 8 : byte;
        if (mine) {
          uint8_t* at = p.scale + row_at * blocks + col0 / 32;
          if (!p.scale_pairs) at[half] = (uint8_t)byte;
          else if (half) *reinterpret_cast<uint16_t*>(at) = (uint16_t)scales;
        }
        if (whole && p.q_rows16) {                       // rows of 64 bytes from both halves
          if (!half) reuse(0);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            *reinterpret_cast<uint4*>(staging + 2048 + lane * 64 + (((2 * half + j) ^ (lane >> 1 & 3)) << 4)) = make_uint4(q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]);
          if (half || left <= 32) send(map_z, 1, col0);
        } else if (mine) {
          store_row8((uint8_t*)p.z + row_at * N + col, q, left, wide);
        }
      }
      if (MODE == GELU_ONLY || MODE == WITH_GELU || MODE == KEEP8) {
#pragma unroll
        for (int j = 0; j < 32; j += 2)
          attn_util::unpack2(quick_gelu2(attn_util::pack2(__float_as_uint(v[j]), __float_as_uint(v[j + 1]))), v[j], v[j + 1]);
      }
      if (GRADIENT) {
        const float scale = act8::value(half ? scales >> 8 : scales & 0xffu);
        const unsigned long long weight2 = attn_util::pack2(__float_as_uint(weight), __float_as_uint(weight));
        unsigned long long dot2 = 0ull;
        uint32_t hw[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float z0, z1, a0, a1;
          if (MODE == GRADIENT8) {
            act8::unpack2(kept[8 * half + (j >> 2)] >> (16 * ((j >> 1) & 1)), scale, &z0, &z1);
          } else {
            z0 = __uint_as_float(kept[16 * half + (j >> 1)] << 16);
            z1 = __uint_as_float(kept[16 * half + (j >> 1)] & 0xffff0000u);
          }
          unsigned long long y, slope;
          quick_gelu_both2(attn_util::pack2(__float_as_uint(z0), __float_as_uint(z1)), &y, &slope);
          const unsigned long long g = attn_util::pack2(__float_as_uint(v[j]), __float_as_uint(v[j + 1]));
          dot2 = attn_util::fma2(g, y, dot2);            // columns behind N: z reads as zero there
          attn_util::unpack2(attn_util::mul2(attn_util::mul2(g, slope), weight2), a0, a1);
          w[j >> 1] = attn_util::pack_bf16(__float_as_uint(a0), __float_as_uint(a1));
          attn_util::unpack2(attn_util::mul2(y, weight2), a0, a1);
          hw[j >> 1] = attn_util::pack_bf16(__float_as_uint(a0), __float_as_uint(a1));
        }
        float a0, a1;
        attn_util::unpack2(dot2, a0, a1);
        dot += a0 + a1;
        if (whole) {
          reuse(1);
          stage(1, hw);
          send(map_z, 1, col);
          reuse(1);
          stage(0, w);
          send(map_y, 0, col);
        } else if (mine) {
          store_row(p.h + row_at * N + col, hw, left, wide);
          store_row(p.y + row_at * N + col, w, left, wide);
        }
        if (mine && p.dots && (half || left <= 32)) p.dots[dots_at(col0 / SLICE, p.rows, row_at)] = dot;
        continue;
      }
      pack_row(v, w);
      if (whole) {
        reuse(MODE == WITH_GELU || (MODE == KEEP8 && p.q_rows16));      // the one store that may be pending is the other buffer's
        stage(0, w);
        send(map_y, 0, col);
      } else if (mine) {
        store_row(p.y + row_at * N + col, w, left, wide);
      }
    }
    return true;
  });
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  if (MODE == PLAIN || MODE == GELU_ONLY || MODE == WITH_GELU) {      // rows behind the last group
    const long long used = group_of(offsets, p.rows, p.experts - 1).r1;
    const long long chunks = (p.rows - used) * (N / 8);
    uint4* rest = reinterpret_cast<uint4*>(p.y + used * N);
    for (long long i = (long long)blockIdx.x * (ROW_GROUPS * 128) + (threadIdx.x - 64); i < chunks; i += (long long)gridDim.x * (ROW_GROUPS * 128))
      rest[i] = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int MODE, bool B_MN>
__global__ void __launch_bounds__(ROW_THREADS, 1)
grouped_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a_few, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_z, const __grid_constant__ CUtensorMap map_kept,
               const __grid_constant__ Problem p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  constexpr int NST = stages_of(MODE);
  Sh* sh = reinterpret_cast<Sh*>(tiles + (size_t)STAGES * STAGE_BYTES + 32768);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = sm100::cluster_ctarank();
  if (warp == 0 && sm100::elect_one()) {
    sm100::tma_prefetch_desc(&map_a);
    sm100::tma_prefetch_desc(&map_b);
    for (int s = 0; s < NST; ++s) { sm100::mbar_init(&sh->full[s], 1); sm100::mbar_init(&sh->empty[s], 1); }
    for (int a = 0; a < 2; ++a) { sm100::mbar_init(&sh->acc_full[a], 1); sm100::mbar_init(&sh->acc_empty[a], 8 * ROW_GROUPS); }
    if (MODE == GRADIENT8 || MODE == GRADIENT16)
      for (int w = 0; w < 4 * ROW_GROUPS; ++w) sm100::mbar_init(&sh->kept[w], 1);
    sh->error = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc_pair(&sh->tmem_base, TMEM_COLS);
    sm100::tmem_relinquish_pair();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();          // the other CTA's barriers exist before anything signals them
  sm100::tc_fence_after();
  const int* offsets = p.offsets;
  const __nv_bfloat16* bias = p.bias;
  const float* row_weights = p.row_weights;
  wait_previous(offsets, bias, row_weights);
  if (!p.offsets) offsets = nullptr;
  if (!p.bias) bias = nullptr;
  if (!p.row_weights) row_weights = nullptr;
  count_tiles(sh, p, offsets, 2 * BM);
  if (warp == 0) {
    if (sm100::elect_one()) produce<NST, B_MN>(sh, tiles, p, offsets, &map_a, &map_a_few, &map_b, rank);
  } else if (warp == 1) {
    if (rank == 0 && sm100::elect_one()) issue<NST, B_MN>(sh, tiles, p, offsets);
  } else {
    finish<MODE>(sh, tiles + (size_t)NST * STAGE_BYTES + (warp - 2) * staging_of(MODE), p, offsets, bias, row_weights, &map_y, &map_z, &map_kept, rank, (warp - 2) >> 2, warp & 3, lane);
  }
  __syncwarp();
  // neither CTA frees its tensor memory or exits while the other may still signal its barriers or have the pair's MMAs read its shared memory
  sm100::tc_fence_before();
  __syncthreads();
  if (sh->error && warp == 0 && sm100::elect_one()) {
    const unsigned long long t0 = sm100::now_ns();
    while (sm100::now_ns() - t0 < 200000000ull) { __nanosleep(1000); }   // copies in flight complete within microseconds
  }
  __syncthreads();
  sm100::cluster_sync();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc_pair(sh->tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- few rows to an expert
// The product the other way round, y^T = w_e x^T, on one CTA per tile: 128 rows of the weight are the M of the MMAs, up to 128 rows of x
// (as many as there are, in steps of 16) their N.  A tile of the kernel above multiplies 256 rows of x whether there are two or 200: with 2
// rows to each of 8 experts, 1024 -> 4096, MMAs were under way for 10 of its 20 us, where the weights need 10.  96 KB of the weights are under way
// per SM.  What bounds this one is the launch with one tile's chain, and then whole rounds of tiles, more than the weights' way from memory: 16 rows, 1024 -> 4096 with a GELU, weights out
// of memory (out of the L2), one expert with rows 7.6 us (6.7), four, 128 tiles, 9.3 (7.6), five, 160 tiles and so a second round, 12.8 (10.3), eight 14.3 (12.0); the bytes
// take 1.3, 5.1, 6.4 and 10.3.
// A thread has a column of y and walks the rows, so a warp's stores are 64 bytes of a row each, the 32 columns of an 8-bit block are its lanes', and a row
// behind the group's end is not touched.
constexpr int FEW_BM = 128, FEW_BN = 128, FEW_STAGES = 6, FEW_EPI_WARPS = 16, FEW_THREADS = 64 + FEW_EPI_WARPS * 32;
constexpr int FEW_A_BYTES = FEW_BM * BK * 2, FEW_STAGE_BYTES = FEW_A_BYTES + FEW_BN * BK * 2;
constexpr size_t FEW_SMEM = (size_t)FEW_STAGES * FEW_STAGE_BYTES + 1024 + 1408;
static_assert(FEW_STAGES == STAGES && FEW_SMEM <= 232448, "shared memory of one CTA");

struct FewUnit { int e, row0, rows, col0, kb0, kb1, slice; };      // first row and rows of x, row of the weight, blocks of K

// f(unit, its number in this CTA's list) for each tile of this CTA until it returns false; the tiles that share a part of the weight follow each other
template <typename F>
__device__ __forceinline__ void for_few(const Sh* sh, const Problem& p, const int* offsets, F f) {
  const int total = sh->tile_end[p.experts - 1], step = (int)gridDim.x;
  int e = 0, it = 0;
  for (int t = (int)blockIdx.x; t < total; t += step, ++it) {
    if (sh->tile_end[e] <= t) {
      int hi = p.experts - 1;
      ++e;
      while (e < hi) {
        const int mid = (e + hi) >> 1;
        if (sh->tile_end[mid] > t) hi = mid;
        else e = mid + 1;
      }
    }
    const int at = t - (e ? sh->tile_end[e - 1] : 0);
    const Group g = group_of(offsets, p.rows, e);
    const int across = (g.r1 - g.r0 + FEW_BN - 1) / FEW_BN, part = at / across;
    FewUnit u;
    u.e = e;
    u.row0 = g.r0 + at % across * FEW_BN;
    u.rows = min(g.r1 - u.row0, FEW_BN);
    u.slice = part % p.slices;
    u.col0 = part / p.slices * FEW_BM;
    u.kb0 = u.slice * p.per;
    u.kb1 = min(p.k_blocks, u.kb0 + p.per);
    if (!f(u, it)) return;
  }
}

__device__ __forceinline__ float one_gelu(float z) {
  float y, none;
  attn_util::unpack2(quick_gelu2(attn_util::pack2(__float_as_uint(z), __float_as_uint(z))), y, none);
  return y;
}

template <int MODE>
__device__ __forceinline__ void few_finish(Sh* sh, const Problem& p, const int* offsets, const __nv_bfloat16* bias_all, const float* row_weights, int group, int quarter, int lane) {
  constexpr bool GRADIENT = MODE == GRADIENT8 || MODE == GRADIENT16;
  const int N = p.N, blocks = (N + 31) / 32;
  for_few(sh, p, offsets, [&](const FewUnit& u, int it) -> bool {
    const int e = u.e, row0 = u.row0, rows = u.rows, col0 = u.col0, acc = it & 1, col = col0 + quarter * 32 + lane;
    const bool in = col < N;
    float* y32 = MODE == PLAIN32 ? p.y32 + (long long)u.slice * p.rows * N : nullptr;
    const float bias = bias_all && in && u.slice == 0 ? __bfloat162float(bias_all[(long long)e * N + col]) : 0.f;
    if (!sm100::mbar_wait_warp(&sh->acc_full[acc], (it >> 1) & 1, kWaitBudgetNs, &sh->error)) { give_up(sh, p.status, 54); return false; }
    sm100::tc_fence_after();
    const uint32_t t_base = sh->tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)acc * FEW_BN;
    // the four groups of warps take 16 rows in turn
    for (int c = group * 16; c < rows && col0 + quarter * 32 < N; c += FEW_EPI_WARPS * 4) {
      const int left = rows - c;
      const long long at0 = (long long)(row0 + c) * N + col;
      uint32_t r[16];
      float z_of[GRADIENT ? 16 : 1], weight_of[GRADIENT ? 16 : 1];
      if (GRADIENT) {                                    // all that these rows need, at once
        uint32_t kept[16], scales[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const bool there = in && j < left;
          const long long row = row0 + c + j, at = at0 + (long long)j * N;
          if (MODE == GRADIENT8) {
            kept[j] = there ? ((const uint8_t*)p.z)[at] : 0u;
            scales[j] = there ? p.scale[row * blocks + col / 32] : 1u;
          } else {
            z_of[j] = there ? __bfloat162float(((const __nv_bfloat16*)p.z)[at]) : 0.f;
          }
          weight_of[j] = row_weights && j < left ? __ldg(row_weights + row) : 1.f;
        }
        if (MODE == GRADIENT8) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float none;
            act8::unpack2(kept[j], act8::value(scales[j]), &z_of[j], &none);
          }
        }
      }
      sm100::tmem_ld_32x16(t_base + c, r);
      sm100::tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (MODE != PLAIN32 && MODE != PLAIN && j >= left) break;
        const long long row = row0 + c + j, at = at0 + (long long)j * N;
        float v = __uint_as_float(r[j]);
        if (!GRADIENT) v += bias;
        if (MODE == PLAIN32) {
          if (in && j < left) y32[at] = v;
        } else if (GRADIENT) {
          const float z = z_of[GRADIENT ? j : 0], weight = weight_of[GRADIENT ? j : 0];
          float y0, y1, d0, d1;
          unsigned long long y, slope;
          quick_gelu_both2(attn_util::pack2(__float_as_uint(z), __float_as_uint(z)), &y, &slope);
          attn_util::unpack2(y, y0, y1);
          attn_util::unpack2(slope, d0, d1);
          if (p.dots) {
            float dot = in ? v * y0 : 0.f;
#pragma unroll
            for (int d = 16; d; d /= 2) dot += __shfl_xor_sync(~0u, dot, d);
            if (lane == 0) p.dots[dots_at(col / 32, p.rows, row)] = dot;
          }
          if (in) {
            p.h[at] = __float2bfloat16_rn(weight * y0);
            p.y[at] = __float2bfloat16_rn(v * d0 * weight);
          }
        } else {
          if (MODE == WITH_GELU && in) ((__nv_bfloat16*)p.z)[at] = __float2bfloat16_rn(v);
          if (MODE == KEEP8) {
            const uint32_t byte = act8::scale_byte(__reduce_max_sync(~0u, in ? act8::magnitude(v) : 0u));
            if (in) ((uint8_t*)p.z)[at] = (uint8_t)act8::pack2(v, 0.f, act8::inverse(byte));
            if (lane == 0) p.scale[row * blocks + col / 32] = (uint8_t)byte;
          }
          if (MODE != PLAIN) v = one_gelu(v);
          if (in && j < left) p.y[at] = __float2bfloat16_rn(v);
        }
      }
    }
    sm100::tc_fence_before();
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive(&sh->acc_empty[acc]);
    return true;
  });
  if (MODE == PLAIN || MODE == GELU_ONLY || MODE == WITH_GELU) {      // rows behind the last group
    const long long used = group_of(offsets, p.rows, p.experts - 1).r1;
    const long long chunks = (p.rows - used) * (N / 8);
    uint4* rest = reinterpret_cast<uint4*>(p.y + used * N);
    for (long long i = (long long)blockIdx.x * (FEW_EPI_WARPS * 32) + (threadIdx.x - 64); i < chunks; i += (long long)gridDim.x * (FEW_EPI_WARPS * 32))
      rest[i] = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int MODE, bool W_MN>
__global__ void __launch_bounds__(FEW_THREADS, 1)
grouped_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_x_half,
                   const __grid_constant__ CUtensorMap map_x_few, const __grid_constant__ Problem p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Sh* sh = reinterpret_cast<Sh*>(tiles + (size_t)FEW_STAGES * FEW_STAGE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0 && sm100::elect_one()) {
    sm100::tma_prefetch_desc(&map_w);
    sm100::tma_prefetch_desc(&map_x);
    for (int s = 0; s < FEW_STAGES; ++s) { sm100::mbar_init(&sh->full[s], 1); sm100::mbar_init(&sh->empty[s], 1); }
    for (int a = 0; a < 2; ++a) { sm100::mbar_init(&sh->acc_full[a], 1); sm100::mbar_init(&sh->acc_empty[a], FEW_EPI_WARPS); }
    sh->error = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc(&sh->tmem_base, 2 * FEW_BN);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const int* offsets = p.offsets;
  const __nv_bfloat16* bias = p.bias;
  const float* row_weights = p.row_weights;
  wait_previous(offsets, bias, row_weights);
  if (!p.offsets) offsets = nullptr;
  if (!p.bias) bias = nullptr;
  if (!p.row_weights) row_weights = nullptr;
  count_tiles(sh, p, offsets, FEW_BN);
  if (warp == 0) {
    if (sm100::elect_one()) {
      Ring ring{0, 0};
      for_few(sh, p, offsets, [&](const FewUnit& u, int) -> bool {
        const int e = u.e, row0 = u.row0, rows = u.rows, col0 = u.col0;
        const CUtensorMap* map = rows > FEW_BN / 2 ? &map_x : rows > FEW ? &map_x_half : &map_x_few;
        const uint32_t tx = FEW_A_BYTES + (rows > FEW_BN / 2 ? FEW_BN : rows > FEW ? FEW_BN / 2 : FEW) * BK * 2;
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          const int stage = ring.stage;
          if (!sm100::mbar_wait(&sh->empty[stage], ring.phase ^ 1, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 51); return false; }
          unsigned char* dst = tiles + (size_t)stage * FEW_STAGE_BYTES;
          sm100::mbar_expect_tx(&sh->full[stage], tx);
          if (!W_MN) {
            sm100::tma_load_3d(dst, &map_w, kb * BK, col0, e, &sh->full[stage]);
          } else {
            sm100::tma_load_3d(dst, &map_w, col0, kb * BK, e, &sh->full[stage]);
            sm100::tma_load_3d(dst + FEW_A_BYTES / 2, &map_w, col0 + 64, kb * BK, e, &sh->full[stage]);
          }
          sm100::tma_load_2d(dst + FEW_A_BYTES, map, kb * BK, row0, &sh->full[stage]);
          advance<FEW_STAGES>(&ring);
        }
        return true;
      });
    }
  } else if (warp == 1) {
    if (sm100::elect_one()) {
      Ring ring{0, 0};
      for_few(sh, p, offsets, [&](const FewUnit& u, int it) -> bool {
        const int acc = it & 1;
        if (!sm100::mbar_wait(&sh->acc_empty[acc], ((it >> 1) & 1) ^ 1, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 52); return false; }
        sm100::tc_fence_after();
        const uint32_t idesc = sm100::make_idesc_f16(FEW_BM, (u.rows + 15) / 16 * 16, true, false, W_MN);
        const uint32_t d = sh->tmem_base + (uint32_t)acc * FEW_BN;
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          const int stage = ring.stage;
          if (!sm100::mbar_wait(&sh->full[stage], ring.phase, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 53); return false; }
          sm100::tc_fence_after();
          const uint32_t a = sm100::smem_u32(tiles + (size_t)stage * FEW_STAGE_BYTES), b = a + FEW_A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t da = W_MN ? sm100::make_desc_sw128_mn(a + k * UMMA_K * 128, FEW_A_BYTES / 2, 1024) : sm100::make_desc_sw128(a + k * UMMA_K * 2);
            sm100::umma_f16(d, da, sm100::make_desc_sw128(b + k * UMMA_K * 2), idesc, (uint32_t)(kb > u.kb0) | (uint32_t)k);
          }
          sm100::umma_commit(&sh->empty[stage]);
          advance<FEW_STAGES>(&ring);
        }
        sm100::umma_commit(&sh->acc_full[acc]);
        return true;
      });
    }
  } else {
    few_finish<MODE>(sh, p, offsets, bias, row_weights, (warp - 2) >> 2, warp & 3, lane);
  }
  __syncwarp();
  sm100::tc_fence_before();
  __syncthreads();
  if (sh->error && warp == 0 && sm100::elect_one()) {
    const unsigned long long t0 = sm100::now_ns();
    while (sm100::now_ns() - t0 < 200000000ull) { __nanosleep(1000); }   // copies in flight complete within microseconds
  }
  __syncthreads();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(sh->tmem_base, 2 * FEW_BN);
  }
}

// ---------------------------------------------------------------- the weights' gradient
struct DwProblem {
  const int* offsets;
  int rows, experts, K, N;   // dw [experts, N, K]
  int bn, tiles_m, tiles_n;  // tiles of 256 rows of N x bn columns of K
  const __nv_bfloat16* dy;   // [rows, N]
  const float* row_weights;  // db_e = sum of row_weights[r] dy_r; null: ones
  __nv_bfloat16* db;         // [experts, N] or null
  int* status;
};

constexpr int EPI_THREADS = ROW_GROUPS * 128;
constexpr int DW_THREADS = ROW_THREADS + 32;            // and the warp that clears rows of other groups
constexpr int DB_GROUPS = EPI_THREADS / (BM / 8);

struct DwSh {
  Shared s;
  uint64_t tail[STAGES];                                // a block with rows of another group: its loads, one barrier per CTA
  uint64_t cleared[STAGES];                             // in the even CTA: the odd one's part of such a block is cleared
};
constexpr int DW_STAGES = 5, DW_STAGING = 4096;           // a warp's 32 rows x 64 columns; the sixth stage's room with the staging
constexpr size_t DW_SMEM = (size_t)DW_STAGES * STAGE_BYTES + 16 * DW_STAGING + 1024 + sizeof(DwSh);
static_assert(DW_SMEM <= 232448 && EPI_THREADS * 8 * 4 <= 16 * DW_STAGING, "shared memory of one CTA");

struct DwUnit { int e, m_blk, n_blk, r0, r1, k_blocks; };

template <typename F>
__device__ __forceinline__ void for_units(const DwProblem& p, const int* offsets, uint32_t rank, F f) {
  const int per = p.tiles_m * p.tiles_n, total = p.experts * per, step = (int)(gridDim.x >> 1);
  for (int t = (int)(blockIdx.x >> 1); t < total; t += step) {
    DwUnit u;
    u.e = t / per;
    int m_tile;
    band_order(t - u.e * per, p.tiles_m, p.tiles_n, &m_tile, &u.n_blk);
    u.m_blk = m_tile * 2 + (int)rank;
    const Group g = group_of(offsets, p.rows, u.e);
    u.r0 = g.r0;
    u.r1 = g.r1;
    u.k_blocks = (g.r1 - g.r0 + BK - 1) / BK;
    if (!f(u)) return;
  }
}

__device__ __forceinline__ void dw_setup(DwSh* sh, int warp, const CUtensorMap* ma, const CUtensorMap* mb) {
  if (warp == 0 && sm100::elect_one()) {
    sm100::tma_prefetch_desc(ma);
    sm100::tma_prefetch_desc(mb);
    for (int s = 0; s < DW_STAGES; ++s) {
      sm100::mbar_init(&sh->s.full[s], 1);
      sm100::mbar_init(&sh->s.empty[s], 1);
      sm100::mbar_init(&sh->tail[s], 1);
      sm100::mbar_init(&sh->cleared[s], 1);
    }
    for (int a = 0; a < 2; ++a) { sm100::mbar_init(&sh->s.acc_full[a], 1); sm100::mbar_init(&sh->s.acc_empty[a], 8 * ROW_GROUPS); }
    sh->s.error = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc_pair(&sh->s.tmem_base, TMEM_COLS);
    sm100::tmem_relinquish_pair();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();
  sm100::tc_fence_after();
}

// One thread in each CTA.
__device__ __forceinline__ void dw_produce(DwSh* shl, unsigned char* tiles, const DwProblem& p, const int* offsets, const CUtensorMap* ma, const CUtensorMap* mb,
                                           uint32_t rank) {
  Shared* sh = &shl->s;
  const int half = p.bn / 2;
  const bool two = half > 64;
  const uint32_t tx = A_BYTES + (two ? B_BYTES : B_BYTES / 2);               // of this CTA
  Ring ring{0, 0};
  for_units(p, offsets, rank, [&](const DwUnit& u) -> bool {
    const int m0 = u.m_blk * BM, n0 = u.n_blk * p.bn + (int)rank * half;
    for (int kb = 0; kb < u.k_blocks; ++kb) {
      const int stage = ring.stage, k0 = u.r0 + kb * BK;
      if (!sm100::mbar_wait(&sh->empty[stage], ring.phase ^ 1, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 41); return false; }
      unsigned char* dst = tiles + (size_t)stage * STAGE_BYTES;
      uint32_t bar = sm100::map_to_cta(&sh->full[stage], 0);
      if (k0 + BK > u.r1) {                             // the clearing warp arrives at full
        bar = sm100::map_to_cta(&shl->tail[stage], rank);
        sm100::mbar_expect_tx(&shl->tail[stage], tx);
      } else if (rank == 0) {
        sm100::mbar_expect_tx(&sh->full[stage], 2 * tx);                       // both CTAs' bytes
      }
      sm100::tma_load_2d_pair(dst, ma, m0, k0, bar);
      sm100::tma_load_2d_pair(dst + A_BYTES / 2, ma, m0 + 64, k0, bar);
      sm100::tma_load_2d_pair(dst + A_BYTES, mb, n0, k0, bar);
      if (two) sm100::tma_load_2d_pair(dst + A_BYTES + B_BYTES / 2, mb, n0 + 64, k0, bar);
      advance<DW_STAGES>(&ring);
    }
    return true;
  });
}

// One warp in each CTA: rows of other groups in the last block of a group become zeros.  A row of 64 elements is 128 bytes at row * 128 of its box, which
// the swizzle permutes within themselves.
__device__ __forceinline__ void dw_clear(DwSh* shl, unsigned char* tiles, const DwProblem& p, const int* offsets, uint32_t rank, int lane) {
  Shared* sh = &shl->s;
  const int boxes = p.bn / 2 > 64 ? 4 : 3;
  int stage = 0;
  uint32_t phases = 0;
  for_units(p, offsets, rank, [&](const DwUnit& u) -> bool {
    const int rem = (u.r1 - u.r0) % BK;
    if (rem) {
      const int at = (stage + u.k_blocks - 1) % DW_STAGES;
      const uint32_t phase = phases >> at & 1;
      if (!sm100::mbar_wait_warp(&shl->tail[at], phase, kWaitBudgetNs, &sh->error)) { give_up(sh, p.status, 45); return false; }
      phases ^= 1u << at;
      unsigned char* box = tiles + (size_t)at * STAGE_BYTES;
      const int upto = (rem + UMMA_K - 1) / UMMA_K * UMMA_K;         // the MMAs read no further
      for (int b = 0; b < boxes; ++b)
        for (int c = rem * 8 + lane; c < upto * 8; c += 32) *reinterpret_cast<uint4*>(box + b * (BK * 128) + c * 16) = make_uint4(0u, 0u, 0u, 0u);
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {                                   // the issuer waits for both
        if (rank) sm100::mbar_arrive_cluster(sm100::map_to_cta(&shl->cleared[at], 0));
        else sm100::mbar_arrive(&sh->full[at]);
      }
    }
    stage = (stage + u.k_blocks) % DW_STAGES;
    return true;
  });
}

// One thread of the even CTA.
__device__ __forceinline__ void dw_issue(DwSh* shl, unsigned char* tiles, const DwProblem& p, const int* offsets) {
  Shared* sh = &shl->s;
  const uint32_t idesc = sm100::make_idesc_f16(2 * BM, p.bn, true, true, true);
  Ring ring{0, 0};
  int it = 0;
  uint32_t cleared = 0;                                  // phases of the barriers of the odd CTA's clearing
  for_units(p, offsets, 0, [&](const DwUnit& u) -> bool {
    if (!u.k_blocks) return true;
    const int acc = it & 1;
    if (!sm100::mbar_wait(&sh->acc_empty[acc], ((it >> 1) & 1) ^ 1, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 42); return false; }
    ++it;
    sm100::tc_fence_after();
    const uint32_t d = sh->tmem_base + (uint32_t)acc * BN;
    for (int kb = 0; kb < u.k_blocks; ++kb) {
      const int stage = ring.stage;
      if (!sm100::mbar_wait(&sh->full[stage], ring.phase, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 43); return false; }
      const int left = u.r1 - u.r0 - kb * BK;
      if (left < BK) {
        if (!sm100::mbar_wait(&shl->cleared[stage], cleared >> stage & 1, kWaitBudgetNs) || sh->error) { give_up(sh, p.status, 46); return false; }
        cleared ^= 1u << stage;
      }
      sm100::tc_fence_after();
      const uint32_t a = sm100::smem_u32(tiles + (size_t)stage * STAGE_BYTES), b = a + A_BYTES;
#pragma unroll
      for (int k = 0; k < BK / UMMA_K; ++k) {
        if (k * UMMA_K >= left) break;
        const uint64_t da = sm100::make_desc_sw128_mn(a + k * UMMA_K * 128, A_BYTES / 2, 1024);
        const uint64_t db = sm100::make_desc_sw128_mn(b + k * UMMA_K * 128, B_BYTES / 2, 1024);
        sm100::umma_f16_pair(d, da, db, idesc, (uint32_t)kb | (uint32_t)k);
      }
      sm100::umma_commit_pair(sm100::map_to_cta(&sh->empty[stage], 0));
      sm100::umma_commit_pair(sm100::map_to_cta(&sh->empty[stage], 1));
      advance<DW_STAGES>(&ring);
    }
    sm100::umma_commit_pair(sm100::map_to_cta(&sh->acc_full[acc], 0));
    sm100::umma_commit_pair(sm100::map_to_cta(&sh->acc_full[acc], 1));
    return true;
  });
}

// whether it holds for all epilogue threads
__device__ __forceinline__ bool all_of(bool ok) {
  uint32_t all;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred q, 3, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(all) : "r"((uint32_t)ok), "n"(EPI_THREADS) : "memory");
  return all != 0;
}
__device__ __forceinline__ void all_sync() { asm volatile("bar.sync 3, %0;" ::"n"(EPI_THREADS) : "memory"); }

// The sums of 128 columns of dY from col0 over the rows [r0, r1), by all epilogue threads; thread `row` of group 0 has column col0 + row.  Thirty-two
// threads share eight columns, each with 16-byte loads of every 32nd row, eight in flight, which are added as a tree; a value passes 3 additions in its batch,
// one for every 256 rows and 5 among the threads.  part: 16 KB of the warps' staging, which their last stores have read.
template <bool WEIGHTS>
__device__ __forceinline__ float column_sums(const DwProblem& p, const __nv_bfloat16* dy, const float* weights, float* part, int col0, int r0, int r1, int group, int row) {
  constexpr int U = 8, STEP = DB_GROUPS;
  const int e = threadIdx.x - 64, col = col0 + (e % (BM / 8)) * 8, mine = e / (BM / 8);
  const int end = col < p.N ? r1 : r0;                  // N is a multiple of 8
  unsigned long long acc[4] = {0ull, 0ull, 0ull, 0ull};                      // two columns each
  for (long long r = (long long)r0 + mine; r < end; r += U * STEP) {
    uint4 v[U];
    float wt[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const bool in = r + i * STEP < end;
      v[i] = in ? __ldcg(reinterpret_cast<const uint4*>(dy + (r + i * STEP) * p.N + col)) : make_uint4(0u, 0u, 0u, 0u);
      if (WEIGHTS) wt[i] = in ? __ldg(weights + r + i * STEP) : 0.f;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      unsigned long long t[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const uint32_t b = w == 0 ? v[i].x : w == 1 ? v[i].y : w == 2 ? v[i].z : v[i].w;
        t[i] = attn_util::pack2(b << 16, b & 0xffff0000u);
        if (WEIGHTS) t[i] = attn_util::mul2(t[i], attn_util::pack2(__float_as_uint(wt[i]), __float_as_uint(wt[i])));
      }
#pragma unroll
      for (int n = U / 2; n; n /= 2)
#pragma unroll
        for (int i = 0; i < n; ++i) t[i] = attn_util::add2(t[i], t[i + n]);
      acc[w] = attn_util::add2(acc[w], t[0]);
    }
  }
  float s[8];
#pragma unroll
  for (int w = 0; w < 4; ++w) attn_util::unpack2(acc[w], s[2 * w], s[2 * w + 1]);
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  all_sync();
  float4* to = reinterpret_cast<float4*>(part + e * 8);
  to[0] = make_float4(s[0], s[1], s[2], s[3]);
  to[1] = make_float4(s[4], s[5], s[6], s[7]);
  all_sync();
  float t[DB_GROUPS];
  if (group == 0) {
#pragma unroll
    for (int g = 0; g < DB_GROUPS; ++g) t[g] = part[g * BM + row];
#pragma unroll
    for (int n = DB_GROUPS / 2; n; n /= 2)
#pragma unroll
      for (int g = 0; g < n; ++g) t[g] += t[g + n];
  }
  all_sync();                          // the staging is the warps' own again
  return group ? 0.f : t[0];
}

__device__ __forceinline__ void dw_finish(DwSh* shl, unsigned char* staging_all, const DwProblem& p, const int* offsets, const CUtensorMap* mdw, const __nv_bfloat16* dy,
                                          const float* row_weights, uint32_t rank, int group, int quarter, int lane) {
  Shared* sh = &shl->s;
  const int row = quarter * 32 + lane, bn = p.bn, c0 = group * SLICE;
  unsigned char* staging = staging_all + ((int)(threadIdx.x >> 5) - 2) * DW_STAGING;
  int it = 0;
  for_units(p, offsets, rank, [&](const DwUnit& u) -> bool {
    const int row0 = u.m_blk * BM, col0 = u.n_blk * bn + c0, warp_row = row0 + quarter * 32;
    if (p.db && u.n_blk == 0) {
      const float sum = row_weights ? column_sums<true>(p, dy, row_weights, reinterpret_cast<float*>(staging_all), row0, u.r0, u.r1, group, row)
                                    : column_sums<false>(p, dy, row_weights, reinterpret_cast<float*>(staging_all), row0, u.r0, u.r1, group, row);
      if (group == 0 && row0 + row < p.N) p.db[(long long)u.e * p.N + row0 + row] = __float2bfloat16_rn(sum);
    }
    const int acc = it & 1;
    if (u.k_blocks) {
      bool ok = sm100::mbar_wait_warp(&sh->acc_full[acc], (it >> 1) & 1, kWaitBudgetNs, &sh->error);
      if (p.db) ok = all_of(ok);                         // where the warps meet for the sums, they go on, or leave, together
      if (!ok) { give_up(sh, p.status, 44); return false; }
      ++it;
      sm100::tc_fence_after();
    }
    const bool busy = c0 < bn && col0 < p.K && warp_row < p.N;
    const uint32_t t_base = sh->tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)acc * BN + c0;
    auto release = [&] {
      if (!u.k_blocks) return;
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive_cluster_no_stores(sm100::map_to_cta(&sh->acc_empty[acc], 0));
    };
    if (!busy) { release(); return true; }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[16];
      if (u.k_blocks) {
        uint32_t r[32];
        sm100::tmem_ld_32x32(t_base + 32 * half, r);
        sm100::tmem_ld_wait();
        if (half) release();
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = attn_util::pack_bf16(r[2 * j], r[2 * j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(staging + lane * 128 + (((4 * half + j) ^ (lane & 7)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    }
    sm100::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      sm100::tma_store_3d(mdw, staging, col0, warp_row, u.e);
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    return true;
  });
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

__global__ void __launch_bounds__(DW_THREADS, 1)
grouped_dw_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_dw,
                  const __grid_constant__ DwProblem p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* staging = tiles + (size_t)DW_STAGES * STAGE_BYTES;
  DwSh* sh = reinterpret_cast<DwSh*>(staging + 16 * DW_STAGING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = sm100::cluster_ctarank();
  dw_setup(sh, warp, &map_dy, &map_x);
  const int* offsets = p.offsets;
  const __nv_bfloat16* dy = p.dy;
  const float* row_weights = p.row_weights;
  wait_previous(offsets, dy, row_weights);
  if (!p.offsets) offsets = nullptr;
  if (!p.row_weights) row_weights = nullptr;
  if (warp == 0) {
    if (sm100::elect_one()) dw_produce(sh, tiles, p, offsets, &map_dy, &map_x, rank);
  } else if (warp == 1) {
    if (rank == 0 && sm100::elect_one()) dw_issue(sh, tiles, p, offsets);
  } else if (warp < 2 + 4 * ROW_GROUPS) {
    dw_finish(sh, staging, p, offsets, &map_dw, dy, row_weights, rank, (warp - 2) >> 2, warp & 3, lane);
  } else {
    dw_clear(sh, tiles, p, offsets, rank, lane);
  }
  __syncwarp();
  teardown(&sh->s, warp);
}

// ---------------------------------------------------------------- host side
// few: grouped_few_kernel
template <int MODE, bool KN>
static const void* kernel_of(bool few) { return few ? (const void*)grouped_few_kernel<MODE, KN> : (const void*)grouped_kernel<MODE, KN>; }
static const void* row_kernel(int mode, bool w_is_kn, bool few) {
  if (w_is_kn)
    return mode == PLAIN32 ? kernel_of<PLAIN32, true>(few) : mode == GRADIENT8 ? kernel_of<GRADIENT8, true>(few)
           : mode == GRADIENT16 ? kernel_of<GRADIENT16, true>(few) : kernel_of<PLAIN, true>(few);
  return mode == GELU_ONLY ? kernel_of<GELU_ONLY, false>(few) : mode == WITH_GELU ? kernel_of<WITH_GELU, false>(few)
         : mode == KEEP8 ? kernel_of<KEEP8, false>(few) : mode == PLAIN32 ? kernel_of<PLAIN32, false>(few) : kernel_of<PLAIN, false>(few);
}

static int max_clusters() {
  static int n = 0;
  static std::once_flag once;
  std::call_once(once, [] {
    for (int mode = PLAIN; mode <= GRADIENT16; ++mode)
      for (int kn = 0; kn < 2; ++kn)
        for (int few = 0; few < 2; ++few)
          cudaFuncSetAttribute(row_kernel(mode, kn != 0, few != 0), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(few ? FEW_SMEM : SMEM));
    cudaFuncSetAttribute((const void*)grouped_dw_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DW_SMEM);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(2 * (gemm_sm_count() / 2)); cfg.blockDim = dim3(DW_THREADS);
    cfg.dynamicSmemBytes = DW_SMEM; cfg.attrs = at; cfg.numAttrs = 1;
    int c = 0;
    if (cudaOccupancyMaxActiveClusters(&c, (void*)grouped_dw_kernel, &cfg) == cudaSuccess && c > 0) n = c;
    else { cudaGetLastError(); n = gemm_sm_count() / 2; }
  });
  return n;
}

// Columns of a tile, for `tiles_m` tiles of rows: whichever takes less time in whole rounds (gemm_pair.cu has the reasons and the costs).
static int tile_columns(long long tiles_m, int N, int clusters) {
  auto cost = [&](int bn, int cycles) { return (tiles_m * ((N + bn - 1) / bn) + clusters - 1) / clusters * cycles; };
  const long long c256 = cost(256, 512), c192 = cost(192, 448), c128 = cost(128, 384);
  if (100 * c128 < 95 * std::min(c256, c192)) return 128;
  return 100 * c192 < 95 * c256 ? 192 : 256;
}

// `clusters` clusters of `size` CTAs
static cudaError_t launch(const void* kernel, long long clusters, int size, int threads, size_t smem, void** args, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // see pdl.cuh
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(size * clusters)); cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem; cfg.stream = stream; cfg.attrs = at; cfg.numAttrs = 2;
  return cudaLaunchKernelExC(&cfg, kernel, args);
}

static int checked(const int* offsets, int rows, int nexperts, int K, int N, const char* what) {
  if (rows < 0 || nexperts < 1 || K < 1 || N < 1) return fail(TMPI_ERR_INVALID, "%s: empty problem", what);
  if (K % 8 || N % 8) return fail(TMPI_ERR_INVALID, "%s: stored rows must be multiples of 16 bytes (TMA)", what);
  if (nexperts > MAX_EXPERTS || (!offsets && nexperts != 1)) return fail(TMPI_ERR_UNSUPPORTED, "%s: at most %d experts", what, MAX_EXPERTS);
  // wrong offsets may ask for this many tiles, which are counted in 32 bits
  if (((long long)rows / (2 * BM) + 1) * nexperts * ((std::max(K, N) + 127) / 128) > 0x7fffffffLL - 2 * BM)
    return fail(TMPI_ERR_UNSUPPORTED, "%s: %d rows, %d experts of %d x %d", what, rows, nexperts, N, K);
  return TMPI_OK;
}

// Rows to an expert, on average, up to which the product is formed the other way round.  Its epilogue takes a row at a time, and longer the more it does.
// us of this form and the other, 8 experts, 1024 -> 4096: GELU with 2 rows each 12.7 and 19.2, 64 12.8 and 20.1, 128 15.7 and 19.5, 160 24.0 and 19.8;
// with a checkpoint, 64 14.6 and 22.9, 160 33.3 and 23.2; the GELU's gradient, 2 13.3 and 21.5, 64 20.6 and 27.3, 96 31.1 and 25.1; 4096 -> 1024
// in fp32, 2 15.2 and 18.7, 128 18.2 and 23.8.  64 ragged groups of 0 to 200 rows, 80 on average, 520 -> 1000: 25.0 and 24.9, with a checkpoint 36.8 and
// 33.5; of half as many, 16.9 and 21.4, with a checkpoint 21.9 and 28.9, the gradient 36.0 and 34.7.
// The host knows the mean alone.  Where few experts have all rows this form is the slower one: 5000 rows of 64 experts, all of one, with a GELU, 520 -> 1000 18.8 and
// 13.5, 1024 -> 4096 44.5 and 33.6; 2048 rows, 2048 <- 512, the GELU's gradient 25 and 15.
static int few_mean(int mode) { return mode == GRADIENT8 || mode == GRADIENT16 ? 32 : mode == KEEP8 ? 64 : 96; }
// Parts of K of a product with few rows and an fp32 result, whose reader adds them: as many as leave eight blocks of K each and about a tile for every SM,
// if half of the experts have rows.  4 tokens with two of 8 experts each, 4096 -> 1024: 14.6 us whole, 9.9 in three parts.
static int few_slices(int rows, int nexperts, int K, int N) {
  if (rows > (long long)few_mean(PLAIN32) * nexperts) return 1;
  const int tiles = std::max(1, std::min(nexperts, rows) / 2 + 1) * ((N + FEW_BM - 1) / FEW_BM), k_blocks = (K + BK - 1) / BK;
  const int most = std::max(1, std::min({4, k_blocks / 8, gemm_sm_count() / tiles}));
  const int per = (k_blocks + most - 1) / most;
  return (k_blocks + per - 1) / per;                    // none is empty
}

static int run(Problem p, const void* x, const void* w, const int* offsets, int rows, int nexperts, int K, int N, bool w_is_kn, int mode, cudaStream_t stream) {
  int st = checked(offsets, rows, nexperts, K, N, "grouped_gemm");
  if (st) return st;
  if (!all_aligned16({x, w, p.bias})) return fail(TMPI_ERR_INVALID, "grouped_gemm: tensors must be 16-byte aligned");
  if (!rows) return TMPI_OK;
  const int clusters = max_clusters();
  p.offsets = offsets; p.rows = rows; p.experts = nexperts; p.K = K; p.N = N;
  p.k_blocks = (K + BK - 1) / BK;
  p.q_rows16 = N % 16 == 0;                              // z itself is on a 16-byte boundary
  p.scale_pairs = N % 64 == 0 && !((uintptr_t)p.scale & 1);
  p.status = gemm_status_word();
  if (rows <= (long long)few_mean(mode) * nexperts) {
    p.slices = mode == PLAIN32 ? few_slices(rows, nexperts, K, N) : 1;
    p.per = (p.k_blocks + p.slices - 1) / p.slices;
    p.tiles_n = (N + FEW_BM - 1) / FEW_BM * p.slices;
    CUtensorMap mw, mx, mx_half, mx_few;
    if (w_is_kn) st = make_tmap_bf16_3d(&mw, w, (uint64_t)nexperts, (uint64_t)K, (uint64_t)N, BK, 64);
    else st = make_tmap_bf16_3d(&mw, w, (uint64_t)nexperts, (uint64_t)N, (uint64_t)K, FEW_BM, 64);
    if (st || (st = make_tmap_bf16(&mx, x, (uint64_t)rows, (uint64_t)K, (uint64_t)K, FEW_BN)) ||
        (st = make_tmap_bf16(&mx_half, x, (uint64_t)rows, (uint64_t)K, (uint64_t)K, FEW_BN / 2)) ||
        (st = make_tmap_bf16(&mx_few, x, (uint64_t)rows, (uint64_t)K, (uint64_t)K, FEW))) return st;
    const long long tiles = ((long long)rows / FEW_BN + std::min(nexperts, rows)) * p.tiles_n;      // at most
    void* args[] = {&mw, &mx, &mx_half, &mx_few, &p};
    const cudaError_t e = launch(row_kernel(mode, w_is_kn, true), std::min<long long>(tiles, gemm_sm_count()), 1, FEW_THREADS, FEW_SMEM, args, stream);
    return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "grouped_gemm launch: %s", cudaGetErrorString(e));
  }
  const long long tiles_m = rows / (2 * BM) + std::min(nexperts, rows);        // at most
  p.bn = tile_columns(tiles_m, N, clusters);
  p.tiles_n = (N + p.bn - 1) / p.bn;
  CUtensorMap ma, ma_few, mb, my, mz, mkept;
  if ((st = make_tmap_bf16(&ma, x, (uint64_t)rows, (uint64_t)K, (uint64_t)K, BM))) return st;
  if ((st = make_tmap_bf16(&ma_few, x, (uint64_t)rows, (uint64_t)K, (uint64_t)K, FEW))) return st;
  if (w_is_kn) st = make_tmap_bf16_3d(&mb, w, (uint64_t)nexperts, (uint64_t)K, (uint64_t)N, BK, 64);
  else st = make_tmap_bf16_3d(&mb, w, (uint64_t)nexperts, (uint64_t)N, (uint64_t)K, p.bn / 2, 64);
  if (st) return st;
  // results go in boxes of 32 rows x 64 bytes (128 in fp32): y, and beside it z, h or the e4m3 numbers
  const bool fp32 = mode == PLAIN32;
  if ((st = make_tmap_box(&my, fp32 ? 4 : 2, fp32 ? (const void*)p.y32 : p.y, (uint64_t)rows, (uint64_t)N, 32, 32))) return st;
  mz = mkept = my;
  if (mode == GRADIENT8 && p.q_rows16) st = make_tmap_box(&mkept, 1, p.z, (uint64_t)rows, (uint64_t)N, 32, 64);
  else if (mode == GRADIENT16) st = make_tmap_box(&mkept, 2, p.z, (uint64_t)rows, (uint64_t)N, 32, 32);
  if (st) return st;
  if (mode == WITH_GELU || mode == GRADIENT8 || mode == GRADIENT16) st = make_tmap_box(&mz, 2, mode == WITH_GELU ? p.z : p.h, (uint64_t)rows, (uint64_t)N, 32, 32);
  else if (mode == KEEP8 && p.q_rows16) st = make_tmap_box(&mz, 1, p.z, (uint64_t)rows, (uint64_t)N, 32, 64);
  if (st) return st;
  void* args[] = {&ma, &ma_few, &mb, &my, &mz, &mkept, &p};
  const cudaError_t e = launch(row_kernel(mode, w_is_kn, false), std::min<long long>(tiles_m * p.tiles_n, clusters), 2, ROW_THREADS, SMEM, args, stream);
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "grouped_gemm launch: %s", cudaGetErrorString(e));
}

}  // namespace grouped
}  // namespace tmpi

using namespace tmpi;

extern "C" {

int tmpi_grouped_max_experts(void) { return grouped::MAX_EXPERTS; }
// the results that tmpi_grouped_gemm leaves in mode 4, [slices, rows, N], whose sum is the product
int tmpi_grouped_slices(int rows, int nexperts, int K, int N) { return rows < 1 || nexperts < 1 || K < 1 || N < 1 ? 1 : grouped::few_slices(rows, nexperts, K, N); }

// y [rows, N] = act(x w_e^T + b_e) for x [rows, K] and w [experts, N, K] (w_is_kn: [experts, K, N], without activation), zeros behind the
// last group; offsets [experts + 1] on the device, or null for one expert.  mode: 0 none; 1 GELU; 2 GELU, and the pre-activation in z; 3 GELU, and
// the pre-activation's 8-bit checkpoint in z and scale [rows, ceil(N / 32)]; 4 none, y in fp32 [tmpi_grouped_slices, rows, N], of which the sum is the
// product, and rows behind the last group left alone.  All bf16
// but those, on 16-byte boundaries (fp32: 32).
int tmpi_grouped_gemm(const void* x, const void* w, const void* bias, const int* offsets, void* y, void* z, void* scale, int rows, int nexperts, int K, int N,
                      int w_is_kn, int mode, void* stream) {
  if (mode < grouped::PLAIN || mode > grouped::PLAIN32 || (w_is_kn && mode && mode != grouped::PLAIN32) ||
      ((mode == grouped::WITH_GELU || mode == grouped::KEEP8) && !z) || (mode == grouped::KEEP8 && !scale))
    return fail(TMPI_ERR_INVALID, "grouped_gemm: mode %d", mode);
  if (!all_aligned16({y, z}) || (mode == grouped::PLAIN32 && (uintptr_t)y % 32)) return fail(TMPI_ERR_INVALID, "grouped_gemm: tensors must be 16-byte aligned");
  grouped::Problem p{};
  p.bias = (const __nv_bfloat16*)bias;
  if (mode == grouped::PLAIN32) p.y32 = (float*)y;
  else p.y = (__nv_bfloat16*)y;
  p.z = z;
  p.scale = (uint8_t*)scale;
  p.wide = N % 32 == 0 && ((uintptr_t)y | (uintptr_t)z) % 32 == 0;
  return grouped::run(p, x, w, offsets, rows, nexperts, K, N, w_is_kn != 0, mode, (cudaStream_t)stream);
}

// the sums of a row that tmpi_grouped_gelu_gradient leaves in dots
int tmpi_grouped_dots(int rows, int nexperts, int N, int kept8) {
  const bool few = rows <= (long long)grouped::few_mean(kept8 ? grouped::GRADIENT8 : grouped::GRADIENT16) * nexperts;
  return few ? (N + 31) / 32 : (N + grouped::SLICE - 1) / grouped::SLICE;
}

// The gradients of gelu(z) h's input and value in one product: with g = dy w_e (dy [rows, K], w [experts, K, N]) in fp32 and the kept z [rows, N] (bf16, or
// with `scale` its 8-bit checkpoint), dz = weight g gelu'(z) and h = weight gelu(z), both bf16 [rows, N]; row_weights fp32 [rows] or null for
// ones.  dots [ceil(tmpi_grouped_dots / 4), rows, 4] (or null): the sums of g gelu(z) over 32 or 64 columns each.  Rows behind the last group are left alone.
int tmpi_grouped_gelu_gradient(const void* dy, const void* w, const int* offsets, const void* z, const void* scale, const float* row_weights, void* dz, void* h,
                               float* dots, int rows, int nexperts, int K, int N, void* stream) {
  if (!all_aligned16({z, dz, h}) || !z || !h) return fail(TMPI_ERR_INVALID, "grouped_gelu_gradient: tensors must be 16-byte aligned");
  grouped::Problem p{};
  p.y = (__nv_bfloat16*)dz;
  p.h = (__nv_bfloat16*)h;
  p.z = const_cast<void*>(z);
  p.scale = (uint8_t*)const_cast<void*>(scale);
  p.row_weights = row_weights;
  p.dots = dots;
  p.wide = N % 32 == 0 && ((uintptr_t)dz | (uintptr_t)h | (uintptr_t)z) % 32 == 0;
  return grouped::run(p, dy, w, offsets, rows, nexperts, K, N, true, scale ? grouped::GRADIENT8 : grouped::GRADIENT16, (cudaStream_t)stream);
}

// dw [experts, N, K] = dy_e^T x_e and, where given, db [experts, N] = the column sums of dy_e, each row times row_weights[row] where given
// (fp32 [rows]); dy [rows, N], x [rows, K], bf16 on 16-byte boundaries.
int tmpi_grouped_weight_gradient(const void* dy, const void* x, const int* offsets, const float* row_weights, void* dw, void* db, int rows, int nexperts, int K,
                                 int N, void* stream) {
  int st = grouped::checked(offsets, rows, nexperts, K, N, "grouped_weight_gradient");
  if (st) return st;
  if (!all_aligned16({dy, x, dw})) return fail(TMPI_ERR_INVALID, "grouped_weight_gradient: tensors must be 16-byte aligned");
  if (!rows) {
    const size_t n = (size_t)nexperts * N;
    cudaError_t e = cudaMemsetAsync(dw, 0, 2 * n * K, (cudaStream_t)stream);
    if (e == cudaSuccess && db) e = cudaMemsetAsync(db, 0, 2 * n, (cudaStream_t)stream);
    return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "grouped_weight_gradient: %s", cudaGetErrorString(e));
  }
  const int clusters = grouped::max_clusters();
  grouped::DwProblem p{};
  p.offsets = offsets; p.rows = rows; p.experts = nexperts; p.K = K; p.N = N;
  p.tiles_m = (N + 2 * gemm2::BM - 1) / (2 * gemm2::BM);
  p.bn = grouped::tile_columns((long long)p.tiles_m * nexperts, K, clusters);
  p.tiles_n = (K + p.bn - 1) / p.bn;
  p.dy = (const __nv_bfloat16*)dy;
  p.row_weights = row_weights;
  p.db = (__nv_bfloat16*)db;
  p.status = gemm_status_word();
  CUtensorMap mdy, mx, mdw;
  if ((st = make_tmap_bf16(&mdy, dy, (uint64_t)rows, (uint64_t)N, (uint64_t)N, gemm2::BK))) return st;
  if ((st = make_tmap_bf16(&mx, x, (uint64_t)rows, (uint64_t)K, (uint64_t)K, gemm2::BK))) return st;
  if ((st = make_tmap_bf16_3d(&mdw, dw, (uint64_t)nexperts, (uint64_t)N, (uint64_t)K, 32, 64))) return st;
  void* args[] = {&mdy, &mx, &mdw, &p};
  const cudaError_t e = grouped::launch((const void*)grouped::grouped_dw_kernel, std::min<long long>((long long)p.tiles_m * p.tiles_n * nexperts, clusters),
                                        2, grouped::DW_THREADS, grouped::DW_SMEM, args, (cudaStream_t)stream);
  return e == cudaSuccess ? TMPI_OK : fail(TMPI_ERR_CUDA, "grouped_weight_gradient launch: %s", cudaGetErrorString(e));
}

}  // extern "C"
