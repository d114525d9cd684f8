// Running sums over the 64 lanes of a wave, in registers: within rows of 16 lanes by shifts, then the last lane of a row added to
// the rows behind it.  (A shuffle goes through LDS: six of them, each waiting for the one before, took 3 times as long.)
#pragma once

#include "common.h"

namespace lh {

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) {  // the other lane's value, 0 where there is none
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp0(uint64_t v) {
  return (uint64_t)dpp0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp0<CTRL, ROWS>((uint32_t)v);
}
// Sum over the lanes up to and with this one (uint32_t or uint64_t).  All 64 lanes take part.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v += dpp0<0x111, 0xf>(v);  // 1, 2, 4, 8 lanes before, within the row
  v += dpp0<0x112, 0xf>(v);
  v += dpp0<0x114, 0xf>(v);
  v += dpp0<0x118, 0xf>(v);
  v += dpp0<0x142, 0xa>(v);  // the last lane of the first and third row, to the row behind
  v += dpp0<0x143, 0xc>(v);  // the last lane of the first half, to the second
  return v;
}
__device__ __forceinline__ uint32_t wave_last(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
__device__ __forceinline__ uint64_t wave_last(uint64_t v) { return (uint64_t)wave_last((uint32_t)(v >> 32)) << 32 | wave_last((uint32_t)v); }
template <typename T>
__device__ __forceinline__ T wave_total(T v) { return wave_last(wave_scan(v)); }

}  // namespace lh
