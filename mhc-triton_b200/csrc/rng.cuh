// Counter-based dropout masks: the keep decision of an element is a function of (seed, offset, row, column)
// alone, so the backward recomputes it and no mask is ever stored.
//
// Generator: Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011), key = seed (64 bits), counter = (column / 8, row, offset low, offset high).  One block of
// 128 bits serves the 8 elements of an aligned group of 8 columns, 16 bits each: element e takes the low (e even)
// or high (e odd) half of word e / 2 and is dropped when that half is below the threshold t, i.e. with
// probability exactly t / 65536; kept elements are scaled by 65536 / (65536 - t), so the expectation is exact
// for the probability used.  16 bits instead of 32 halve the cost, which is what a bf16 tensor can afford at
// memory speed: ten rounds are 20 32x32->64-bit multiplications per 8 elements.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mhc {

struct Drop {
  const int64_t* rng;  // device: {seed, offset}
  uint32_t thr;        // dropped when u16 < thr; 1 .. 65535
  float scale;         // 65536 / (65536 - thr)
  uint32_t row0;       // added to the row index
};

struct DropKey { uint32_t k0, k1, c2, c3; };

__device__ __forceinline__ DropKey drop_key(const Drop& d) {
  const uint64_t seed = (uint64_t)__ldg((const unsigned long long*)d.rng);
  const uint64_t off = (uint64_t)__ldg((const unsigned long long*)d.rng + 1);
  return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

__device__ __forceinline__ uint4 philox4x32_10(const DropKey& key, uint32_t col8, uint32_t row) {
  uint32_t c0 = col8, c1 = row, c2 = key.c2, c3 = key.c3, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The random halves of the V columns from `col` on (V = 8 or 4: col is a multiple of V; V = 1: any).
template <int V> struct DropBits { uint32_t w[V > 1 ? V / 2 : 1]; };

template <int V>
__device__ __forceinline__ DropBits<V> drop_bits(const Drop& d, const DropKey& key, int64_t row, int64_t col) {
  const uint4 r = philox4x32_10(key, (uint32_t)(col >> 3), (uint32_t)row + d.row0);
  DropBits<V> o;
  if constexpr (V == 1) {  // the half the column owns, in the upper half of the word
    const int e = (int)(col & 7);
    const uint32_t lo = (e & 2) ? r.y : r.x, hi = (e & 2) ? r.w : r.z;
    const uint32_t w = (e & 4) ? hi : lo;
    o.w[0] = (e & 1) ? w : w << 16;
  } else if constexpr (V == 4) {
    const bool up = (col & 4) != 0;
    o.w[0] = up ? r.z : r.x;
    o.w[1] = up ? r.w : r.y;
  } else {
    static_assert(V == 8, "pack width");
    o.w[0] = r.x; o.w[1] = r.y; o.w[2] = r.z; o.w[3] = r.w;
  }
  return o;
}

// v[e] -> 0 where dropped (whatever v held, infinities and NaN included), v * scale where kept.
template <int V>
__device__ __forceinline__ void drop_apply(const Drop& d, const DropBits<V>& b, float (&v)[V]) {
  const uint32_t t = d.thr << 16;
#pragma unroll
  for (int e = 0; e < V; ++e) {  // u16 >= thr, compared in the upper half of a word
    const uint32_t u = V == 1 ? b.w[0] : (e & 1) ? b.w[e >> 1] : b.w[e >> 1] << 16;
    v[e] = u >= t ? v[e] * d.scale : 0.f;
  }
}

}  // namespace mhc
