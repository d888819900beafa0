// integer_exp (integer_lut.rs:56-74) in 32 bits from a table in shared memory
// that holds each entry beside the step to the next: one 8-byte lookup.
#pragma once
#include "lut.cuh"

__device__ __forceinline__ void load_lut(int2* lut, int nt) {
  for (int i = threadIdx.x; i < q16::EXP_LUT_N; i += nt) {
    const int lo = (int)g_exp_lut.v[i];
    lut[i] = make_int2(lo, i < q16::EXP_LUT_N - 1 ? (int)g_exp_lut.v[i + 1] - lo : 0);
  }
}
// x > 0 counts as 0.
__device__ __forceinline__ int exp32(int x, const int2* lut) {
  const int off = min(max(x + (int)q16::EXP_RANGE, 0), (int)q16::EXP_RANGE);
  const int2 t = lut[off >> 11];
  return off > 0 ? t.x + ((t.y * (off & 2047)) >> 11) : 0;
}
