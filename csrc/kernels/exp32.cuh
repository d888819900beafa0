// integer_exp (integer_lut.rs:56-74) in 32 bits from a table in shared memory.
//
// For off = x + EXP_RANGE > 0 the value is lo + ((step * (off mod 2^11)) >> 11)
// with lo and step of segment off >> 11; for off <= 0 it is 0.  Counted from 1,
// off - 1 = 2^11 k + f, it is (lo_k 2^11 + step_k (f + 1)) >> 11 in segment k
// (at the segment's end the next entry, as it must be).  Entry k + 1 holds
// (lo_k 2^11 + step_k, step_k), entry 0 zeros: with the sum clamped from below
// to entry 0's last place, one add-and-max, one 8-byte lookup, one product and
// one shift.
#pragma once
#include "lut.cuh"

constexpr int EXP_TABLE_N = 512;  // 257 used; the index has 9 bits, whatever x is
constexpr int EXP_AT = (int)q16::EXP_RANGE + 2047;

__device__ __forceinline__ int2 exp_entry(int i) {
  const int lo = i ? (int)g_exp_lut.v[i - 1] : 0, step = i ? (int)g_exp_lut.v[i] - lo : 0;
  return make_int2((lo << 11) + step, step);
}
__device__ __forceinline__ void load_exp(int2* table, int nt) {
  for (int i = threadIdx.x; i < q16::EXP_LUT_N; i += nt) table[i] = exp_entry(i);
}
// at = max(x + EXP_AT, 2047) with x <= 0; anything for x > 0, without a fault.
__device__ __forceinline__ uint32_t exp_at(int at, const int2* table) {
  const int2 t = *(const int2*)((const uint8_t*)table + (at >> 8 & 0xff8));
  return (uint32_t)(t.x + t.y * (at & 2047)) >> 11;
}
// The exp of x + (at - EXP_AT).
__device__ __forceinline__ uint32_t exp32(int x, int at, const int2* table) {
  return exp_at(__viaddmax_s32(x, at, 2047), table);
}
