// Two fp32 operations in one instruction (each rounded on its own, as if done singly): half the issue slots of the
// element-wise arithmetic.  The pack functions apply them to a whole pack; single elements stay single.  What it gives shows in
// long runs, where the power cap holds the clock: add + norm forward + backward at 32768 x 4096 bf16 380 -> 372 us, the stream
// form at 2 x 4096 x 4096 168 -> 161, e4m3 output at 16384 x 7168 145 -> 141.  The dropout's scaling gains nothing from it.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mhc {

__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// a[e] *= f
template <int V> __device__ __forceinline__ void pack_scale(float (&a)[V], float f) {
  if constexpr (V == 1) {
    a[0] *= f;
  } else {
    const uint64_t ff = pair(f, f);
#pragma unroll
    for (int e = 0; e < V; e += 2) unpair(mul2(pair(a[e], a[e + 1]), ff), a[e], a[e + 1]);
  }
}
// a[e] *= b[e]
template <int V> __device__ __forceinline__ void pack_mul(float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    a[0] *= b[0];
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) unpair(mul2(pair(a[e], a[e + 1]), pair(b[e], b[e + 1])), a[e], a[e + 1]);
  }
}
// a[e] += b[e]
template <int V> __device__ __forceinline__ void pack_add(float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    a[0] += b[0];
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) unpair(add2(pair(a[e], a[e + 1]), pair(b[e], b[e + 1])), a[e], a[e + 1]);
  }
}
// c[e] += a[e] b[e]
template <int V> __device__ __forceinline__ void pack_fma(float (&c)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    c[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2)
      unpair(fma2(pair(a[e], a[e + 1]), pair(b[e], b[e + 1]), pair(c[e], c[e + 1])), c[e], c[e + 1]);
  }
}
// a[e] = a[e] b[e] + c[e]
template <int V> __device__ __forceinline__ void pack_mul_add(float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) {
    a[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2)
      unpair(fma2(pair(a[e], a[e + 1]), pair(b[e], b[e + 1]), pair(c[e], c[e + 1])), a[e], a[e + 1]);
  }
}
// Sum of a[e] b[e] beside `sum`: two running sums, kept apart until the row's end.
struct Sum2 { uint64_t s; };
template <int V> __device__ __forceinline__ void pack_dot(Sum2& sum, const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    float lo, hi;
    unpair(sum.s, lo, hi);
    sum.s = pair(fmaf(a[0], b[0], lo), hi);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) sum.s = fma2(pair(a[e], a[e + 1]), pair(b[e], b[e + 1]), sum.s);
  }
}
__device__ __forceinline__ float total(const Sum2& sum) {
  float a, b;
  unpair(sum.s, a, b);
  return a + b;
}

}  // namespace mhc
