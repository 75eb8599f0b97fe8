// hif4_enc.cuh -- pieces of the HiF4 encoders shared by the codec and the
// key/value cache (files compiled with -fmad=false).
#pragma once
#include "common.cuh"
#include "log2_floor_table.h"

namespace hif4x {

// floor(torch.log2(t)) for finite t > 0.
__device__ __forceinline__ int floor_log2_torch(float t) {
  const uint32_t b = __float_as_uint(t);
  int e = (int)(b >> 23) - 127;
  if ((b >> 23) == 0) e = (31 - __clz((int)b)) - 149;
  e = min(e, HIF4X_LOG2_EMAX);
  return e + (b >= HIF4X_LOG2_UP[e - HIF4X_LOG2_EMIN] ? 1 : 0);
}

// E6M2 code of a scale: (E + 48) << 2 | M
__device__ __forceinline__ uint32_t e6m2_code(float sf) {
  const uint32_t b = __float_as_uint(sf);
  const int E = (int)(b >> 23) - 127;
  return ((uint32_t)(E + 48) << 2) | ((b >> 21) & 3u);
}

// ---- packed fp32 pairs (sm_100 f32x2 arithmetic, round-to-nearest per lane)
typedef unsigned long long u64;
__device__ __forceinline__ u64 pk2(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void upk2(u64 v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ u64 sub2(u64 a, u64 b) {
  u64 d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

}  // namespace hif4x
