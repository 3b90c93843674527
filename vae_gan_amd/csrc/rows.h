// What the row operators share: column folds (norm.hip) and reductions over a wave.
#pragma once
#include "common.h"

// out[col] = sum_p part[p][cols] in a fixed order; columns below `split` go to out0, the others to out1 (either may be
// null).  Outputs are rounded once to `dtype`.
int vg_fold_cols(const float* part, int parts, int64_t cols, void* out0, int64_t split, void* out1, int dtype, hipStream_t st);

// Sum / maximum over the 64 lanes, the same in every lane: adds along rows of 16 lanes and from row to row in registers
// (a shuffle goes through LDS and takes some 60 cycles a step; these take the ALU's own).
template <int CTRL, int ROWS> __device__ __forceinline__ float wave_move(float old, float v) {
  return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp((int)__float_as_uint(old), (int)__float_as_uint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_last(float v) { return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63)); }
__device__ __forceinline__ float wave_sum64(float v) {
  v += wave_move<0x111, 0xf>(0.f, v);                // lane i takes lane i - 1, then - 2, - 4, - 8 within its row
  v += wave_move<0x112, 0xf>(0.f, v);
  v += wave_move<0x114, 0xf>(0.f, v);
  v += wave_move<0x118, 0xf>(0.f, v);
  v += wave_move<0x142, 0xa>(0.f, v);                // rows 1 and 3 take the last lane of the row before
  v += wave_move<0x143, 0xc>(0.f, v);                // rows 2 and 3 take lane 31
  return wave_last(v);
}
__device__ __forceinline__ float wave_max64(float v) {
  v = fmaxf(v, wave_move<0x111, 0xf>(v, v));
  v = fmaxf(v, wave_move<0x112, 0xf>(v, v));
  v = fmaxf(v, wave_move<0x114, 0xf>(v, v));
  v = fmaxf(v, wave_move<0x118, 0xf>(v, v));
  v = fmaxf(v, wave_move<0x142, 0xa>(v, v));
  v = fmaxf(v, wave_move<0x143, 0xc>(v, v));
  return wave_last(v);
}
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned wave_umax_step(unsigned v) {
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xf, false);
  return o > v ? o : v;
}
__device__ __forceinline__ unsigned wave_umax64(unsigned v) {
  v = wave_umax_step<0x111, 0xf>(v);
  v = wave_umax_step<0x112, 0xf>(v);
  v = wave_umax_step<0x114, 0xf>(v);
  v = wave_umax_step<0x118, 0xf>(v);
  v = wave_umax_step<0x142, 0xa>(v);
  v = wave_umax_step<0x143, 0xc>(v);
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
