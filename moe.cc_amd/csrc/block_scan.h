// block_scan.h - sums over the threads of a block, for whole numbers.
#pragma once
#include "moe_device.h"

namespace moe {

// Sum over a block of N threads up to and without this one, and of all.  wave_s: N / 64 numbers in LDS.
template <int N>
__device__ __forceinline__ int block_scan(int v, int* wave_s, int* total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int x = v;
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  if (lane == kWave - 1) wave_s[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < N / kWave; ++w) {
    const int y = wave_s[w];
    if (w < wave) before += y;
    all += y;
  }
  __syncthreads();
  *total = all;
  return before + x - v;
}

}  // namespace moe
