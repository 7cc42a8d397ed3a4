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

// The ten rounds, split by what they depend on.  With the counter (column / 8, row, offset) the multiplications of
// rounds 1 to 3 depend on the column or on the row alone: a thread that stays in its columns and walks rows does the
// column's part once (DropCol), the row's single multiplication once per row (DropRow), and 15 of the 20
// multiplications per block.
struct DropSeed { uint32_t k0, k1, row_x, c1, c3; };  // row_x, c1: what round 1 makes of the offset's low word
struct DropCol { uint32_t x, y, z, c3; };
struct DropRow { uint32_t hi, lo; };

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u, kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;

// A value that is the same in all lanes, as one the compiler knows to be: the sums with the round constants then leave the
// vector pipes (the dropout of 32768 x 4096 bf16 went from 138 us to 110 by this alone; with its rows and CTAs as they are in
// dropout.cu it takes 92).  Whole warps only.
__device__ __forceinline__ uint32_t warp_uniform(uint32_t v) { return __reduce_or_sync(0xffffffffu, v); }

// Called by whole warps.
__device__ __forceinline__ DropSeed drop_seed(const Drop& d) {
  uint64_t seed = (uint64_t)__ldg((const unsigned long long*)d.rng);
  uint64_t off = (uint64_t)__ldg((const unsigned long long*)d.rng + 1);
  seed = ((uint64_t)warp_uniform((uint32_t)(seed >> 32)) << 32) | warp_uniform((uint32_t)seed);
  off = ((uint64_t)warp_uniform((uint32_t)(off >> 32)) << 32) | warp_uniform((uint32_t)off);
  const uint64_t b = (uint64_t)(uint32_t)off * kPhiloxM1;
  DropSeed s;
  s.k0 = (uint32_t)seed;
  s.k1 = (uint32_t)(seed >> 32);
  s.row_x = (uint32_t)(b >> 32) ^ s.k0;
  s.c1 = (uint32_t)b;
  s.c3 = (uint32_t)(off >> 32);
  return s;
}

__device__ __forceinline__ DropCol drop_col(const DropSeed& s, uint32_t col8) {
  const uint64_t a1 = (uint64_t)col8 * kPhiloxM0;                               // round 1
  const uint64_t b2 = (uint64_t)((uint32_t)(a1 >> 32) ^ s.c3 ^ s.k1) * kPhiloxM1;  // round 2
  const uint64_t a3 = (uint64_t)((uint32_t)(b2 >> 32) ^ s.c1 ^ (s.k0 + kPhiloxW0)) * kPhiloxM0;  // round 3
  DropCol c;
  c.x = (uint32_t)a1 ^ (s.k1 + kPhiloxW1);
  c.y = (uint32_t)b2 ^ (s.k0 + 2 * kPhiloxW0);
  c.z = (uint32_t)(a3 >> 32) ^ (s.k1 + 2 * kPhiloxW1);
  c.c3 = (uint32_t)a3;
  return c;
}

__device__ __forceinline__ DropRow drop_row(const Drop& d, const DropSeed& s, int64_t row) {
  const uint64_t a2 = (uint64_t)(s.row_x ^ ((uint32_t)row + d.row0)) * kPhiloxM0;  // round 2
  return DropRow{(uint32_t)(a2 >> 32), (uint32_t)a2};
}

__device__ __forceinline__ uint4 drop_block(const DropSeed& s, const DropCol& col, const DropRow& row) {
  const uint64_t b3 = (uint64_t)(row.hi ^ col.x) * kPhiloxM1;                   // round 3
  uint32_t c0 = (uint32_t)(b3 >> 32) ^ col.y, c1 = (uint32_t)b3, c2 = col.z ^ row.lo, c3 = col.c3;
#pragma unroll
  for (int i = 3; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * kPhiloxM0, b = (uint64_t)c2 * kPhiloxM1;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ (s.k0 + (uint32_t)i * kPhiloxW0);
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ (s.k1 + (uint32_t)i * kPhiloxW1);
    c3 = (uint32_t)a;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The random halves of the V columns from `col` on (V = 8 or 4: col is a multiple of V; V = 1: any).
template <int V> struct DropBits { uint32_t w[V > 1 ? V / 2 : 1]; };

template <int V>
__device__ __forceinline__ DropBits<V> drop_bits(const DropSeed& s, const DropCol& dc, const DropRow& dr, int64_t col) {
  const uint4 r = drop_block(s, dc, dr);
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

// The bits of a thread that stays in the V columns from `col` on and walks the rows row, row + step, ...  With single
// columns the 8 lanes of a group of columns each compute the block of one of the next 8 rows and hand the words round:
// one block per 8 elements, as with packs.  The warp must walk together then, lanes past the last column included.
template <int V> struct DropWalk {
  DropSeed seed;
  DropCol col;
  uint4 block;
  int used;
  __device__ __forceinline__ void start(const DropSeed& s, int64_t c0) {
    seed = s;
    col = drop_col(s, (uint32_t)(c0 >> 3));
    used = 8;
  }
  __device__ __forceinline__ DropBits<V> bits(const Drop& d, int64_t row, int64_t step, int64_t c0) {
    if constexpr (V > 1) {
      return drop_bits<V>(seed, col, drop_row(d, seed, row), c0);
    } else {
      const int lane = threadIdx.x & 31;
      if (used == 8) {
        block = drop_block(seed, col, drop_row(d, seed, row + (lane & 7) * step));
        used = 0;
      }
      const int from = (lane & 24) | used++;
      const uint32_t x = __shfl_sync(0xffffffffu, block.x, from), y = __shfl_sync(0xffffffffu, block.y, from);
      const uint32_t z = __shfl_sync(0xffffffffu, block.z, from), w = __shfl_sync(0xffffffffu, block.w, from);
      const uint32_t lo = (lane & 2) ? y : x, hi = (lane & 2) ? w : z, word = (lane & 4) ? hi : lo;
      DropBits<1> o;
      o.w[0] = (lane & 1) ? word : word << 16;
      return o;
    }
  }
};

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
