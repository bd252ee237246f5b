// Two fp32 numbers that one instruction works on.
#pragma once

#include <cuda_runtime.h>

namespace rmn {

struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair make_pair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ void parts(Pair p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p.v)); }
__device__ __forceinline__ Pair add(Pair a, Pair b) {
  Pair p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return p;
}
__device__ __forceinline__ float total(Pair a) {
  float x, y;
  parts(a, x, y);
  return x + y;
}

}  // namespace rmn
