// The rows of rank numbers that a projection takes as more K (adapter.cu makes them, adapter_tcgen05.cu too;
// gemm_rows_tcgen05.cu and gemm_tcgen05_pair.cu read them).
//
// A tensor-core product of bfloat16 operands would round a rank number to 8 bits. It goes there as two numbers,
// u = hi + lo with hi = bf16(u) and lo = bf16(u - hi): 16 bits, 2^-16 of it left out at most, and all of it where it
// has no more bits. Both meet the same B, so that their two products are the same sum's.
//
// A K block of 64 columns has 32 ranks: their hi halves, then their lo ones; the ranks behind the last one are
// zeros. B is read as it is stored, 32 of its columns a block, and both halves' instructions take those. (The halves
// in K blocks of their own would be as many blocks for ranks of whole 64, and one more of each adapter
// for ranks up to 32.)
#pragma once

#include <cuda_bf16.h>

constexpr int FB_PLANE_RANKS = 32;

// Ranks of a row, those behind the last one included, and its bfloat16 numbers.
__host__ __device__ constexpr int fb_plane_ranks(int rank) {
  return (rank + FB_PLANE_RANKS - 1) / FB_PLANE_RANKS * FB_PLANE_RANKS;
}
__host__ __device__ constexpr int fb_plane_width(int rank) { return 2 * fb_plane_ranks(rank); }

// Rank j's number into its row. (A number that rounds to infinity has no second half, which would be its negative.)
__device__ __forceinline__ void fb_store_halves(__nv_bfloat16* row, int j, float u) {
  __nv_bfloat16* to = row + j / FB_PLANE_RANKS * 2 * FB_PLANE_RANKS + j % FB_PLANE_RANKS;
  const __nv_bfloat16 hi = __float2bfloat16_rn(u);
  const float whole = __bfloat162float(hi);
  to[0] = hi;
  to[FB_PLANE_RANKS] = __float2bfloat16_rn(isinf(whole) ? 0.f : u - whole);
}
