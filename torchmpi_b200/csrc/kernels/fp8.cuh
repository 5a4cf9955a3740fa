// A matrix in 8 bits with a scale for each block of 128: 128 consecutive elements of a row share a power of two 2^e, and each is kept as
// e4m3(x / 2^e).  The exponent is chosen as for the 8-bit checkpoints (act8.cuh): the smallest from -126 under which the block's largest
// finite magnitude is at most 448; a value is rounded once, by at most half an e4m3 step, infinities and NaN become NaN.
//
// A power of two, because the tensor cores multiply by it themselves (tcgen05.mma with block scales takes a byte e + 127 for each row
// and 32 elements of K): products of blocks go into one fp32 accumulator, where scales of any value would have to be applied to each
// block's sums apart, on their way out of tensor memory.
//
// The numbers lie in rows of a pitch that is a multiple of 128, zeros behind the last column.  The scales lie as the tensor cores read them: 512 bytes
// for 128 rows x 4 blocks, row r and block b of those at (r % 32) * 16 + r / 32 * 4 + b, the tiles of a row of tiles one after another.
#pragma once
#include "act8.cuh"

namespace tmpi {
namespace fp8 {

constexpr int BLOCK = 128, TILE_ROWS = 128, GROUP = 4, TILE_BYTES = TILE_ROWS * GROUP;

__host__ __device__ __forceinline__ int blocks_of(long long cols) { return (int)((cols + BLOCK - 1) / BLOCK); }
__host__ __device__ __forceinline__ int groups_of(long long cols) { return (blocks_of(cols) + GROUP - 1) / GROUP; }
__host__ __device__ __forceinline__ long long pitch_of(long long cols) { return (long long)blocks_of(cols) * BLOCK; }

// where the scale of row r, block b lies
__device__ __forceinline__ size_t scale_at(long long r, int b, int groups) {
  const int in = (int)(r & (TILE_ROWS - 1));
  return ((size_t)(r >> 7) * groups + (b >> 2)) * TILE_BYTES + (in & 31) * 16 + (in >> 5) * 4 + (b & 3);
}

}  // namespace fp8
}  // namespace tmpi
