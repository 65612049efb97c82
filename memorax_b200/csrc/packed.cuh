// Two floats in a register pair: sm_100a adds, multiplies and fuses both in one instruction (each rounded as by itself), which
// is what streaming kernels that are short of issue slots need.
#pragma once

#include <stdint.h>

namespace mxk {

struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2() = default;
  __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ explicit F2(float both) : F2(both, both) {}
  __device__ __forceinline__ float lo() const { float a, b; asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); return a; }
  __device__ __forceinline__ float hi() const { float a, b; asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); return b; }
  __device__ __forceinline__ F2 swapped() const { return F2(hi(), lo()); }
  __device__ __forceinline__ float sum() const { return lo() + hi(); }
};
__device__ __forceinline__ F2 add(F2 a, F2 b) { F2 c; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v)); return c; }
__device__ __forceinline__ F2 sub(F2 a, F2 b) { F2 c; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v)); return c; }
__device__ __forceinline__ F2 mul(F2 a, F2 b) { F2 c; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v)); return c; }
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) { F2 d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return d; }

}  // namespace mxk
