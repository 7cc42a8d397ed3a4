// Root-mean-square norm of the rows a sub-layer reads, with what surrounds it fused in:
//   s    = x (+ residual), x optionally through the counter-based dropout of rng.cuh     (Src::Add)
//        = sum_n H_pre[n] H[n], the mix of the four streams                              (Src::Mix)
//   rstd = 1 / sqrt(mean(s^2) + eps),  y = s * rstd * weight
// y leaves in the activation type, or as e4m3 with one scale per row or per group of 32 / 64 / 128 columns.
// Backward: with c = sum_d dy w s,  ds = rstd (dy w - s rstd^2 c / D) (+ the gradient that reached s directly),
// dweight = sum_rows dy s rstd; dropout's mask is recomputed.  All sums, the norm and the scales are fp32.  s is
// normalised as computed, before it is rounded to the activation type for sum_out, and the backward forms it again
// from x and residual instead of reading the rounded sum_out: one more tensor to read (5 instead of 4 of a bf16
// backward's moves), but dweight keeps fp32 accuracy (from the rounded sums it is off by 1e-3).  It is a sum in fp32 over the
// rows a CTA walks and in fp64 above that: off by 1.3e-7 of the columns' root mean square in the median and 8e-7 at most at
// 32768 x 4096 bf16 (fp64 throughout: 4e-8 and 2.6e-7; the row's own roundings).  Where the mix is
// stored as branch_input, the stored value is what is normalised, so its backward, which reads it, is exact too.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "launch.h"
#include "pairs.cuh"
#include "rng.cuh"

namespace mhc {

enum class Src { Add, Mix };
enum class Out { Plain, RowScale, GroupScale };

constexpr float kE4m3Max = 448.f;
constexpr float kMinScale = 1.17549435082228751e-38f;  // 2^-126: keeps 1 / scale finite for rows of zeros

struct NormFwd {
  const void* x;         // [rows, D], or H [rows, 4, D]
  const void* res;       // [rows, D] or null
  const float* hpre;     // [B, 4] (Mix)
  const void* weight;    // [D] or null (ones)
  int w_f32;             // weight is fp32 (else: the activation type)
  void* sum_out;         // [rows, D] or null
  void* y;               // [rows, D] activation type, or e4m3 bytes
  void* scales;          // [rows, G] fp32 or e8m0 bytes
  float* rstd;           // [rows] or null
  int64_t rows, S, D;
  int group, shift;      // columns per scale (GroupScale): 1 << shift
  int G;                 // scales per row
  int scales8;           // e8m0 scales of 32 columns, 8 at a time on 8 bytes
  int e8m0;
  float eps;
  float inv_D;
  float inv_D_lo;        // 1 / D = inv_D + inv_D_lo
  Drop drop;
};

struct NormBwd {
  const void* dy;        // [rows, D]
  const void* dsum;      // [rows, D] or null: gradient that reaches s beside the norm
  const void* x;         // [rows, D], or H [rows, 4, D]
  const void* res;       // [rows, D] or null
  const float* hpre;
  const float* rstd;     // [rows]
  const void* weight;
  int w_f32;
  void* dx;              // [rows, D], or dH [rows, 4, D]
  void* dres;            // [rows, D] or null (dropout: the gradient before the mask)
  float* dw_part;        // [ctas, D] or null
  float* dpre_part;      // [B, chunks, 4] (Mix)
  int64_t items, S, D;   // items: rows (Add), batch elements x chunks (Mix)
  int parts;             // rows of dw_part
  int64_t chunks;        // per batch element (Mix)
  float inv_D;
  Drop drop;
};

template <typename T, int V> __device__ __forceinline__ void unpack(const RawPack<T, V>& r, float (&o)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = raw_get<V>(r, e);
}

template <typename T> __device__ __forceinline__ float load_w(const void* w, int w_f32, int64_t d) {
  if (!w) return 1.f;
  return w_f32 ? __ldg((const float*)w + d) : to_f32(__ldg((const T*)w + d));
}

// max that keeps NaN (fmaxf drops it): a row that holds one must not get a finite scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// 1 / sqrt(mean + eps) from a sum of squares: the hardware's approximation (2^-22.9) and one Newton step.
__device__ __forceinline__ float row_rstd(float ss, float inv_D, float eps) {
  const float x = fmaf(ss, inv_D, eps), r = rsqrtf(x);
  return x > 1e-30f && x < 1e30f ? fmaf(0.5f * r, fmaf(-x * r, r, 1.f), r) : r;   // elsewhere the step itself would lose
}
// The same to about 45 bits, as hi + lo, for 8-bit outputs, where an error of the last fp32 bit moves a value or a
// power-of-two scale that is next to a border to the other side (1 scale in 4 million at 16384 x 7168).  Products and
// their exact errors by FMA; in fp64 it cost 9 us of 133 at that shape.
struct Rstd2 { float hi, lo; };
__device__ __forceinline__ Rstd2 row_rstd2(float ss, float inv_hi, float inv_lo, float eps) {
  const float p = ss * inv_hi, pe = fmaf(ss, inv_hi, -p) + ss * inv_lo;   // mean = p + pe
  const float x = p + eps, big = fmaxf(p, eps), small = fminf(p, eps);
  const float xe = (big - x + small) + pe;                                // x + xe = mean + eps
  Rstd2 r;
  r.hi = rsqrtf(x);
  const float t = x * r.hi, te = fmaf(x, r.hi, -t) + xe * r.hi;           // (x + xe) hi
  const float e = fmaf(-t, r.hi, 1.f) - te * r.hi;                        // 1 - (x + xe) hi^2
  r.lo = x > 1e-30f && x < 1e30f ? 0.5f * r.hi * e : 0.f;
  return r;
}

// Scale of the values u rstd whose largest |u| is `umax`, and the two factors that take u itself to e4m3.
// fp32: scale = umax rstd / 448 and u (448 / umax): rstd cancels, so a quotient is two roundings from s w.
// e8m0: the next power of two that is not below the largest |value| / 448 (so nothing saturates), as its biased
// exponent: 448 = 1.75 * 2^8, so that is the value's exponent - 8, plus one if its mantissa is above 1.75, which the
// carry of an integer addition says exactly; NaN and infinity become the NaN code 255.
struct Scale { float f1, f2, f32; uint32_t code; };
__device__ __forceinline__ Scale make_scale(float umax, const Rstd2& rstd, int e8m0) {
  Scale r;
  r.f1 = rstd.hi + rstd.lo;
  const float amax = fmaf(umax, rstd.hi, umax * rstd.lo);
  if (e8m0) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)((b + 0x1fffffu) >> 23) - 8;
    const bool finite = b < 0x7f800000u;
    r.code = finite ? (uint32_t)(e < 1 ? 1 : e) : 255u;
    r.f32 = 0.f;   // not stored
    r.f2 = finite ? __uint_as_float((254u - r.code) << 23) : __int_as_float(0x7fc00000);
  } else {
    const float s = __fdiv_rn(amax, kE4m3Max);
    r.code = 0;
    if (s < kMinScale) {  // false for NaN
      r.f32 = kMinScale;
      r.f2 = 8.50705917302346159e37f;   // 2^126
    } else if (umax < 1.2e-35f) {   // 448 / umax could overflow where rstd is large; amax is not below 448 * 2^-126
      r.f32 = s;
      r.f2 = __fdiv_rn(kE4m3Max, amax);
    } else {
      r.f32 = s;
      r.f1 = __fdiv_rn(kE4m3Max, umax);
      r.f2 = 1.f;
    }
  }
  return r;
}

__device__ __forceinline__ void store_scale(void* scales, int64_t i, const Scale& s, int e8m0) {
  if (e8m0) ((uint8_t*)scales)[i] = (uint8_t)s.code;
  else ((float*)scales)[i] = s.f32;
}

// Sum (and NaN-keeping maximum) over a CTA; the result reaches every thread.  Fixed order.
template <bool MAX>
__device__ __forceinline__ void block_sum_max(float& sum, float& mx, float* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (MAX) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    sm[warp] = sum;
    if (MAX) sm[32 + warp] = mx;
  }
  __syncthreads();
  float t = 0.f, m = 0.f;
  for (int w = 0; w < nw; ++w) {
    t += sm[w];
    if (MAX) m = max_nan(m, sm[32 + w]);
  }
  sum = t;
  mx = m;
}

// ------------------------------------------ rows too wide for registers (16-bit types over 16384 columns; fp32, odd or
// unaligned ones over 8192).  Read element by element, twice, and dweight is updated in memory: right, not fast.  4096 x 32768
// bf16 with a residual 484 us forward (164 at the memory's rate) and 2548 backward (205); fp32 4096 x 16384 270 and 925.
// s[row, d], read element by element.
template <typename T, Src SRC, bool DROP>
__device__ __forceinline__ float src_at(const NormFwd& a, const DropSeed& seed, const float (&pre)[4], int64_t row, int64_t d) {
  if constexpr (SRC == Src::Mix) {
    const T* h = (const T*)a.x + row * 4 * a.D + d;
    const float b = ((pre[0] * to_f32(__ldg(h)) + pre[1] * to_f32(__ldg(h + a.D))) + pre[2] * to_f32(__ldg(h + 2 * a.D))) +
                    pre[3] * to_f32(__ldg(h + 3 * a.D));
    return a.sum_out ? to_f32(from_f32<T>(b)) : b;
  } else {
    float v[1] = {to_f32(__ldg((const T*)a.x + row * a.D + d))};
    if constexpr (DROP) drop_apply<1>(a.drop, drop_bits<1>(seed, drop_col(seed, (uint32_t)(d >> 3)), drop_row(a.drop, seed, row), d), v);
    if (a.res) v[0] += to_f32(__ldg((const T*)a.res + row * a.D + d));
    return v[0];
  }
}

// One CTA of 256 threads per row; the row is read again for every pass over it.
template <typename T, Src SRC, bool DROP, Out OUT>
__global__ void __launch_bounds__(256)
k_norm_any_fwd(NormFwd a) {
  pdl_prologue();
  __shared__ float sm[64];
  const int64_t row = blockIdx.x, D = a.D;
  float pre[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (SRC == Src::Mix) {
#pragma unroll
    for (int n = 0; n < 4; ++n) pre[n] = __ldg(a.hpre + row / a.S * 4 + n);
  }
  DropSeed seed{};
  if constexpr (DROP) seed = drop_seed(a.drop);
  float ss = 0.f, mx = 0.f;
  for (int64_t d = threadIdx.x; d < D; d += 256) {
    const float v = src_at<T, SRC, DROP>(a, seed, pre, row, d);
    if (a.sum_out) ((T*)a.sum_out)[row * D + d] = from_f32<T>(v);
    ss = fmaf(v, v, ss);
    if (OUT == Out::RowScale) mx = max_nan(mx, fabsf(v * load_w<T>(a.weight, a.w_f32, d)));
  }
  block_sum_max<OUT == Out::RowScale>(ss, mx, sm);
  if constexpr (OUT == Out::Plain) {
    const float rstd = row_rstd(ss, a.inv_D, a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    for (int64_t d = threadIdx.x; d < D; d += 256)
      ((T*)a.y)[row * D + d] =
          from_f32<T>(src_at<T, SRC, DROP>(a, seed, pre, row, d) * rstd * load_w<T>(a.weight, a.w_f32, d));
  } else if constexpr (OUT == Out::RowScale) {
    const Scale s = make_scale(mx, row_rstd2(ss, a.inv_D, a.inv_D_lo, a.eps), a.e8m0);
    if (threadIdx.x == 0) store_scale(a.scales, row, s, a.e8m0);
    for (int64_t d = threadIdx.x; d < D; d += 256) {
      const float u = src_at<T, SRC, DROP>(a, seed, pre, row, d) * load_w<T>(a.weight, a.w_f32, d);
      ((uint8_t*)a.y)[row * D + d] = (uint8_t)e4m3x2(u * s.f1 * s.f2, 0.f);
    }
  } else {  // a warp per group
    const Rstd2 rstd = row_rstd2(ss, a.inv_D, a.inv_D_lo, a.eps);
    const int64_t G = a.G;
    const int lane = threadIdx.x & 31;
    for (int64_t g = threadIdx.x >> 5; g < G; g += 8) {
      float y[4], m = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t d = g * a.group + j * 32 + lane;
        y[j] = 0.f;
        if (j * 32 < a.group && d < D)
          y[j] = src_at<T, SRC, DROP>(a, seed, pre, row, d) * load_w<T>(a.weight, a.w_f32, d);
        m = max_nan(m, fabsf(y[j]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      const Scale s = make_scale(m, rstd, a.e8m0);
      if (lane == 0) store_scale(a.scales, row * G + g, s, a.e8m0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t d = g * a.group + j * 32 + lane;
        if (j * 32 < a.group && d < D) ((uint8_t*)a.y)[row * D + d] = (uint8_t)e4m3x2(y[j] * s.f1 * s.f2, 0.f);
      }
    }
  }
}

// Persistent CTAs of 256 threads: CTA i takes items i, i + grid, ...  An item is a row (Add), or a share of the tokens of
// one batch element (Mix), whose dH_pre it sums (block_store_f64).  dweight's partial sums live in the CTA's own row of dw_part.
template <typename T, Src SRC, bool DROP>
__global__ void __launch_bounds__(256)
k_norm_any_bwd(NormBwd a) {
  pdl_prologue();
  __shared__ float sm[64];
  __shared__ double red[8 * 4];
  const int64_t D = a.D;
  DropSeed seed{};
  if constexpr (DROP) seed = drop_seed(a.drop);
  float* dw = a.dw_part ? a.dw_part + (int64_t)blockIdx.x * D : nullptr;
  if (dw)
    for (int64_t d = threadIdx.x; d < D; d += 256) dw[d] = 0.f;
  for (int64_t it = blockIdx.x; it < a.items; it += gridDim.x) {
    int64_t r0 = it, r1 = it + 1;   // RowMap of this kernel: one row at a time
    float pre[4] = {0.f, 0.f, 0.f, 0.f};
    double dpre[4] = {0.0, 0.0, 0.0, 0.0};
    if constexpr (SRC == Src::Mix) {
      const int64_t b = it / a.chunks;
      r0 = b * a.S + it % a.chunks;
      r1 = (b + 1) * a.S;
#pragma unroll
      for (int n = 0; n < 4; ++n) pre[n] = __ldg(a.hpre + b * 4 + n);
    }
    for (int64_t row = r0; row < r1; row += SRC == Src::Mix ? a.chunks : 1) {
      const float rstd = __ldg(a.rstd + row);
      NormFwd f;
      f.x = a.x; f.res = a.res; f.sum_out = nullptr; f.D = D; f.drop = a.drop;
      auto s_at = [&](int64_t d) -> float { return src_at<T, SRC, DROP>(f, seed, pre, row, d); };
      float c = 0.f, unused = 0.f;
      for (int64_t d = threadIdx.x; d < D; d += 256) {
        const float dy = to_f32(__ldg((const T*)a.dy + row * D + d)), s = s_at(d);
        c = fmaf(dy * load_w<T>(a.weight, a.w_f32, d), s, c);
        if (dw) dw[d] = fmaf(dy, s * rstd, dw[d]);
      }
      __syncthreads();  // the previous row's readers of sm are done
      block_sum_max<false>(c, unused, sm);
      const float k = c * rstd * rstd * rstd * a.inv_D;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int64_t d = threadIdx.x; d < D; d += 256) {
        const float dy = to_f32(__ldg((const T*)a.dy + row * D + d));
        float g[1] = {rstd * (dy * load_w<T>(a.weight, a.w_f32, d)) - s_at(d) * k};
        if constexpr (SRC == Src::Mix) {
          const T* h = (const T*)a.x + row * 4 * D + d;
          T* o = (T*)a.dx + row * 4 * D + d;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            acc[n] = fmaf(g[0], to_f32(__ldg(h + n * D)), acc[n]);
            o[n * D] = from_f32<T>(pre[n] * g[0]);
          }
        } else {
          if (a.dsum) g[0] += to_f32(__ldg((const T*)a.dsum + row * D + d));
          if constexpr (DROP) {
            if (a.dres) ((T*)a.dres)[row * D + d] = from_f32<T>(g[0]);
            drop_apply<1>(a.drop, drop_bits<1>(seed, drop_col(seed, (uint32_t)(d >> 3)), drop_row(a.drop, seed, row), d), g);
          }
          ((T*)a.dx)[row * D + d] = from_f32<T>(g[0]);
        }
      }
      if constexpr (SRC == Src::Mix) {
#pragma unroll
        for (int n = 0; n < 4; ++n) dpre[n] += (double)acc[n];
      }
    }
    if constexpr (SRC == Src::Mix) {
      __syncthreads();
      block_store_f64(dpre, a.dpre_part + it * 4, red);
    }
  }
}

// --------------------------------------------------------------------------------------------- rows held in registers
// A row belongs to `tpr` threads (a multiple of 32) that own NP packs each, all loaded before the first use and kept in
// registers as fp32 between the row sum and the output, so the data is read once.  Narrow rows share a CTA of 256
// threads.  Bound by memory; the one barrier of a row is covered by the other CTAs.
// Rows that do not divide into packs (odd widths, unaligned tensors) use the same kernels with packs of one element.
struct RowMap {
  int tpr;   // threads per row
  int rpc;   // rows per CTA
  int DV;    // packs per row
};

// The packs of thread t of a row: first, first + step, ...  Wide packs are spread over the row; single elements stay
// within the warp's own 32 NP columns, whose dropout bits and groups of 64 or 128 columns are then the warp's affair.
template <int V, int NP> struct Packs {
  int first, step;
  __device__ __forceinline__ Packs(int t, const RowMap& m)
      : first(V > 1 ? t : (t >> 5) * 32 * NP + (t & 31)), step(V > 1 ? m.tpr : 32) {}
};

template <typename T, int V> __device__ __forceinline__ RawPack<T, V> raw_zero() {
  RawPack<T, V> r;
  if constexpr (V == 1) r.w = from_f32<T>(0.f);
  else r.w = make_uint4(0, 0, 0, 0);
  return r;
}

// Dropout bits of the thread's packs in one row.  With single elements a lane computes the block of one of the warp's 32
// groups of 8 columns (NP = 8) and the warp exchanges the halves through 512 bytes of shared memory of its own.
template <int V, int NP>
__device__ __forceinline__ void drop_row_bits(const DropSeed& seed, const DropCol (&dcol)[V > 1 ? NP : 1], const DropRow& drow,
                                              const Packs<V, NP>& pk, uint4* exchange, DropBits<V> (&bits)[NP]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int k = 0; k < NP; ++k) bits[k] = drop_bits<V>(seed, dcol[k], drow, (pk.first + k * pk.step) * V);
  } else {
    static_assert(NP == 8, "one block per lane");
    uint4* mine = exchange + (threadIdx.x >> 5) * 32;
    __syncwarp();
    mine[threadIdx.x & 31] = drop_block(seed, dcol[0], drow);
    __syncwarp();
    const uint16_t* h = reinterpret_cast<const uint16_t*>(mine) + (threadIdx.x & 31);
#pragma unroll
    for (int k = 0; k < NP; ++k) bits[k].w[0] = (uint32_t)h[k * 32] << 16;
  }
}
template <int V, int NP>
__device__ __forceinline__ void drop_cols(const DropSeed& seed, const Packs<V, NP>& pk, int t, DropCol (&dcol)[V > 1 ? NP : 1]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int k = 0; k < NP; ++k) dcol[k] = drop_col(seed, (uint32_t)((pk.first + k * pk.step) * V) >> 3);
  } else {
    dcol[0] = drop_col(seed, (uint32_t)t);   // t-th group of 8 columns of the row
  }
}

// Row sum (and NaN-keeping maximum) over the warps of one row; sm holds 2 x 32 floats.  One barrier.
template <bool MAX>
__device__ __forceinline__ void row_sum_max(float& sum, float& mx, float* sm, const RowMap& m, int sub) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (MAX) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (m.tpr == 32) return;
  const int warp = threadIdx.x >> 5, nw = m.tpr >> 5, l = threadIdx.x & 31;
  if ((threadIdx.x & 31) == 0) {
    sm[warp] = sum;
    if (MAX) sm[32 + warp] = mx;
  }
  __syncthreads();
  sum = l < nw ? sm[sub * nw + l] : 0.f;
  if (MAX) mx = l < nw ? sm[32 + sub * nw + l] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (MAX) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_w_pack(const void* w, int w_f32, int col, float (&o)[V]) {
  if constexpr (V == 1) {
    o[0] = load_w<T>(w, w_f32, col);
  } else if (!w) {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 1.f;
  } else if (w_f32) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>((const float*)w + col + e));
      o[e] = f.x; o[e + 1] = f.y; o[e + 2] = f.z; o[e + 3] = f.w;
    }
  } else {
    RawPack<T, V> r;
    r.w = __ldg(reinterpret_cast<const uint4*>((const T*)w + col));
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = raw_get<V>(r, e);
  }
}

template <int V> __device__ __forceinline__ void store_e4m3(uint8_t* p, float (&u)[V], float f) {
  pack_scale<V>(u, f);
  if constexpr (V == 1) {
    *p = (uint8_t)e4m3x2(u[0], 0.f);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = (uint32_t)e4m3x2(u[4 * i], u[4 * i + 1]) | ((uint32_t)e4m3x2(u[4 * i + 2], u[4 * i + 3]) << 16);
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// From a row's values v (fp32; v w for an 8-bit output), its sum of squares and, for a scale per row, its largest |v w| to the
// output: finishes the sums over the row's threads (a barrier), then normalises, scales and stores.  `at` is the element
// offset of the thread's first pack, DV the row's packs (0: the row does not exist).
template <typename T, int V, int NP, Out OUT>
__device__ __forceinline__ void norm_emit(const NormFwd& a, const RowMap& m, const Packs<V, NP>& pk, float* sm, int sub, int t,
                                          int DV, int64_t row, int64_t at, float (&v)[NP][V], const float (&w)[NP][V],
                                          float ss, float mx) {
  const int stride = pk.step * V;
  row_sum_max<OUT == Out::RowScale>(ss, mx, sm, m, sub);
  if constexpr (OUT == Out::Plain) {
    const float rstd = row_rstd(ss, a.inv_D, a.eps);
    if (a.rstd && DV && t == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      pack_scale<V>(v[k], rstd);
      pack_mul<V>(v[k], w[k]);
      if (pk.first + k * pk.step < DV) PackIO<T, V>::store((T*)a.y + at + k * stride, v[k]);
    }
  } else {
    const Rstd2 rstd = row_rstd2(ss, a.inv_D, a.inv_D_lo, a.eps);
    Scale sc{};
    float g[NP];   // largest |v w| of the group a pack is in
    if constexpr (OUT == Out::RowScale) {
      sc = make_scale(mx, rstd, a.e8m0);
      if (DV && t == 0) store_scale(a.scales, row, sc, a.e8m0);
    }
    if constexpr (OUT == Out::GroupScale) {
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        g[k] = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) g[k] = max_nan(g[k], fabsf(v[k][e]));
      }
    }
    if constexpr (OUT == Out::GroupScale && V == 1) {   // 64 or 128 columns are 2 or 4 consecutive k of the warp
#pragma unroll
      for (int k = 0; k < NP; k += 2)
        if (a.group >= 64) g[k] = g[k + 1] = max_nan(g[k], g[k + 1]);
#pragma unroll
      for (int k = 0; k < NP; k += 4)
        if (a.group >= 128) g[k] = g[k + 1] = g[k + 2] = g[k + 3] = max_nan(g[k], g[k + 2]);
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int p = pk.first + k * pk.step;
      if constexpr (OUT == Out::GroupScale) {
        // group / V consecutive lanes share it (V = 1: the warp)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          if (V == 1 || o * V < 32 || o * V < a.group) g[k] = max_nan(g[k], __shfl_xor_sync(0xffffffffu, g[k], o));
        sc = make_scale(g[k], rstd, a.e8m0);
        if (V == 8 && a.scales8) {   // a warp's 8 scales as one store: one by one the bytes cost 10 us of 142
          const int lane = threadIdx.x & 31;
          const uint32_t c = (p < DV && (lane & 3) == 0) ? sc.code << (8 * ((lane >> 2) & 3)) : 0u;
          const uint32_t lo = __reduce_or_sync(0xffffffffu, lane < 16 ? c : 0u);
          const uint32_t hi = __reduce_or_sync(0xffffffffu, lane < 16 ? 0u : c);
          if (p < DV && lane == 0)
            *reinterpret_cast<uint2*>((uint8_t*)a.scales + row * a.G + (p >> 2)) = make_uint2(lo, hi);
        } else if (p < DV && (p * V & (a.group - 1)) == 0) {
          store_scale(a.scales, row * a.G + (p * V >> a.shift), sc, a.e8m0);
        }
      }
      pack_scale<V>(v[k], sc.f1);
      if (p < DV) store_e4m3<V>((uint8_t*)a.y + at + k * stride, v[k], sc.f2);
    }
  }
}

// Adds up a pack's squares; for an 8-bit output v becomes v w, whose largest magnitude a scale per row needs.
template <int V, Out OUT>
__device__ __forceinline__ void norm_gather(float (&v)[V], const float (&w)[V], Sum2& ss, float& mx) {
  pack_dot<V>(ss, v, v);
  if (OUT != Out::Plain) pack_mul<V>(v, w);
  if (OUT == Out::RowScale) {
#pragma unroll
    for (int e = 0; e < V; ++e) mx = max_nan(mx, fabsf(v[e]));
  }
}

template <typename T, int V>
__device__ __forceinline__ void mix_pack(const RawPack<T, V> (&x)[4], const float (&pre)[4], float (&v)[V]) {
  float u[V];
  unpack<T, V>(x[0], v);
  pack_scale<V>(v, pre[0]);
#pragma unroll
  for (int n = 1; n < 4; ++n) {
    const float p[2] = {pre[n], pre[n]};
    unpack<T, V>(x[n], u);
    if constexpr (V == 1) {
      v[0] = fmaf(p[0], u[0], v[0]);
    } else {
#pragma unroll
      for (int e = 0; e < V; e += 2) unpair(fma2(pair(p[0], p[1]), pair(u[e], u[e + 1]), pair(v[e], v[e + 1])), v[e], v[e + 1]);
    }
  }
}

// One row per thread group, once: bound by memory (162 us at 32768 x 4096 bf16 with a residual and the sum written, four
// tensors = 6.6 TB/s), for the many CTAs an SM holds and their short lives; a persistent form of it took 176.
template <typename T, int V, int NP, Src SRC, bool DROP, Out OUT>
__global__ void __launch_bounds__(V == 1 ? 1024 : 512, NP == 2 ? 2 : 1)
k_norm_fwd(NormFwd a, RowMap m) {
  pdl_prologue();
  __shared__ float sm[64];
  __shared__ uint4 exchange[DROP && V == 1 ? 1024 : 1];
  const int sub = m.rpc == 1 ? 0 : threadIdx.x / m.tpr, t = threadIdx.x - sub * m.tpr;
  const Packs<V, NP> pk(t, m);
  const int64_t row = (int64_t)blockIdx.x * m.rpc + sub, D = a.D, at = row * D + pk.first * V;
  const int DV = row < a.rows ? m.DV : 0, stride = pk.step * V;   // a row past the end owns no packs
  constexpr int NS = SRC == Src::Mix ? 4 : 2;
  const T* xp = (const T*)a.x + (SRC == Src::Mix ? 4 : 1) * row * D + pk.first * V;
  const T* rp = (const T*)a.res + at;
  RawPack<T, V> raw[NP][NS];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
#pragma unroll
    for (int n = 0; n < NS; ++n) raw[k][n] = raw_zero<T, V>();
    if (pk.first + k * pk.step < DV) {
      if constexpr (SRC == Src::Mix) {
#pragma unroll
        for (int n = 0; n < 4; ++n) raw[k][n] = ld_raw<T, V>(xp + n * D + k * stride);
      } else {
        raw[k][0] = ld_raw<T, V>(xp + k * stride);
        if (a.res) raw[k][1] = ld_raw<T, V>(rp + k * stride);
      }
    }
  }
  float pre[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (SRC == Src::Mix) {
    if (DV) {
      const float* h = a.hpre + (int64_t)((uint32_t)row / (uint32_t)a.S) * 4;   // at most 2^31 rows, four weights each
#pragma unroll
      for (int n = 0; n < 4; ++n) pre[n] = __ldg(h + n);
    }
  }
  float w[NP][V];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
#pragma unroll
    for (int e = 0; e < V; ++e) w[k][e] = 0.f;
    if (pk.first + k * pk.step < DV) load_w_pack<T, V>(a.weight, a.w_f32, pk.first * V + k * stride, w[k]);
  }
  DropBits<V> bits[NP];
  if constexpr (DROP) {
    const DropSeed seed = drop_seed(a.drop);
    DropCol dcol[V > 1 ? NP : 1];
    drop_cols<V, NP>(seed, pk, t, dcol);
    drop_row_bits<V, NP>(seed, dcol, drop_row(a.drop, seed, row), pk, exchange, bits);
  }
  T* so = (T*)a.sum_out + at;
  float v[NP][V], mx = 0.f;
  Sum2 ss{0};
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const bool ok = pk.first + k * pk.step < DV;
    if constexpr (SRC == Src::Mix) {
      mix_pack<T, V>(raw[k], pre, v[k]);
      if (a.sum_out && ok) PackIO<T, V>::store_round(so + k * stride, v[k]);
    } else {
      unpack<T, V>(raw[k][0], v[k]);
      if constexpr (DROP) drop_apply<V>(a.drop, bits[k], v[k]);
      if (a.res) {
        float u[V];
        unpack<T, V>(raw[k][1], u);
        pack_add<V>(v[k], u);
      }
      if (a.sum_out && ok) PackIO<T, V>::store(so + k * stride, v[k]);
    }
    norm_gather<V, OUT>(v[k], w[k], ss, mx);
  }
  norm_emit<T, V, NP, OUT>(a, m, pk, sm, sub, t, DV, row, at, v, w, total(ss), mx);
}

// Many rows and more to do per pack than to add, norm and store it (8-bit output, dropout): persistent CTAs that keep the
// weight and the columns' part of the generator in registers, with the next row's packs on the way by cp.async into slots of
// shared memory that only the thread itself reads.  The one-shot form is bound by instructions there: 16384 x 7168 bf16 to
// e4m3 with a scale per 32 columns 170 us against 132-137 (6.0-6.2 TB/s), 8192 x 7168 with dropout 90 against 81.
template <typename T, int V, int NP, Src SRC, bool DROP, Out OUT>
__global__ void __launch_bounds__(512, 2)
k_norm_fwd_ring(NormFwd a, RowMap m) {
  extern __shared__ __align__(16) uint4 ring[];   // [2][NP][NS][threads]
  __shared__ float sm[2][64];
  pdl_prologue();
  constexpr int NS = SRC == Src::Mix ? 4 : 2;
  const int sub = m.rpc == 1 ? 0 : threadIdx.x / m.tpr, t = threadIdx.x - sub * m.tpr;
  const Packs<V, NP> pk(t, m);
  const int64_t D = a.D;
  const int stride = pk.step * V;
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16u, pitch = blockDim.x * 16u;
  const uint32_t rows = (uint32_t)a.rows, step = gridDim.x * m.rpc;   // at most 2^31 rows
  auto issue = [&](int stage, uint32_t row) {
    if (row < rows) {
      const T* xp = (const T*)a.x + (SRC == Src::Mix ? 4 : 1) * (int64_t)row * D + t * V;
      const T* rp = (const T*)a.res + (int64_t)row * D + t * V;
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (t + k * m.tpr < m.DV) {
#pragma unroll
          for (int n = 0; n < NS; ++n)
            if (SRC == Src::Mix || n == 0 || a.res)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + (uint32_t)((stage * NP + k) * NS + n) * pitch),
                           "l"((SRC == Src::Mix ? xp + n * D : n == 0 ? xp : rp) + k * stride)
                           : "memory");
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto slot = [&](int stage, int k, int n) -> RawPack<T, V> {
    RawPack<T, V> r;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.w.x), "=r"(r.w.y), "=r"(r.w.z), "=r"(r.w.w)
                 : "r"(mine + (uint32_t)((stage * NP + k) * NS + n) * pitch)
                 : "memory");
    return r;
  };
  uint32_t row = blockIdx.x * m.rpc + sub;
  issue(0, row);
  DropSeed seed{};
  DropCol dcol[NP];
  float w[NP][V];
  if constexpr (DROP) drop_cols<V, NP>(seed = drop_seed(a.drop), pk, t, dcol);
#pragma unroll
  for (int k = 0; k < NP; ++k) {
#pragma unroll
    for (int e = 0; e < V; ++e) w[k][e] = 0.f;
    if (t + k * m.tpr < m.DV) load_w_pack<T, V>(a.weight, a.w_f32, t * V + k * stride, w[k]);
  }
  int stage = 0;
  for (uint32_t base = blockIdx.x * m.rpc; base < rows; base += step, row += step) {   // uniform over the CTA
    issue(stage ^ 1, row + step);
    const int DV = row < rows ? m.DV : 0;
    const int64_t at = (int64_t)row * D + t * V;
    float pre[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (SRC == Src::Mix) {
      if (DV) {
        const float* h = a.hpre + (int64_t)(row / (uint32_t)a.S) * 4;
#pragma unroll
        for (int n = 0; n < 4; ++n) pre[n] = __ldg(h + n);
      }
    }
    DropBits<V> bits[NP];
    if constexpr (DROP)   // while the row is on its way
      drop_row_bits<V, NP>(seed, dcol, drop_row(a.drop, seed, row), pk, nullptr, bits);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    float v[NP][V], mx = 0.f;
    Sum2 ss{0};
#pragma unroll
    for (int k = 0; k < NP; ++k) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[k][e] = 0.f;
      if (t + k * m.tpr < DV) {
        if constexpr (SRC == Src::Mix) {
          RawPack<T, V> x[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) x[n] = slot(stage, k, n);
          mix_pack<T, V>(x, pre, v[k]);
          if (a.sum_out) PackIO<T, V>::store_round((T*)a.sum_out + at + k * stride, v[k]);
        } else {
          unpack<T, V>(slot(stage, k, 0), v[k]);
          if constexpr (DROP) drop_apply<V>(a.drop, bits[k], v[k]);
          if (a.res) {
            float u[V];
            unpack<T, V>(slot(stage, k, 1), u);
            pack_add<V>(v[k], u);
          }
          if (a.sum_out) PackIO<T, V>::store((T*)a.sum_out + at + k * stride, v[k]);
        }
        norm_gather<V, OUT>(v[k], w[k], ss, mx);
      }
    }
    norm_emit<T, V, NP, OUT>(a, m, pk, sm[stage], sub, t, DV, row, at, v, w, total(ss), mx);
    stage ^= 1;   // the next row's sums go to the other half of sm: nobody can still be reading it
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Backward: persistent CTAs, so that the threads, which own the same columns in every row, keep the weight and
// dweight's running sums in registers.  The packs of the next DEPTH - 1 rows are on the way meanwhile, by cp.async into
// slots of shared memory that only the thread itself reads (no barrier): in registers they spilled, and the
// stream form ran at 42 % of the memory's rate.  An item is rpc rows (Add) or one of `chunks` shares of a batch element's
// tokens (Mix): every chunks-th group of rpc tokens, so that the CTAs sweep the memory side by side.  DEPTH 0 (single
// elements, which cp.async cannot copy): loads straight from memory.  204 us at 32768 x 4096 bf16 (five tensors, 6.6 TB/s),
// 118 at 8192 x 7168 with dropout (six, 6.0 TB/s, bound by instructions: 14 warps per SM and twice as many per pack), 108
// for the streams at 2 x 4096 x 4096 (nine, 5.6 TB/s).  One pack per thread and twice the warps was no faster.
// Two instances have more values than registers and spill: four packs of 16-bit values per thread (rows of 8193 to 16384 columns;
// 216 bytes of stores, 472 for the streams, 660 with dropout; 273 us at 8192 x 16384 bf16, 205 at the memory's rate, 443
// with dropout, 258 for the streams at 2 x 2048 x 16384, 185) and single elements in more than 512 threads (4097 to 8192 columns;
// 248, 456 for the streams; 272 us at 8192 x 6001 bf16, 75 at the memory's rate).
template <typename T, int V, int NP, int DEPTH, int THREADS, Src SRC, bool DROP>
__global__ void __launch_bounds__(THREADS)
k_norm_bwd(NormBwd a, RowMap m) {
  extern __shared__ __align__(16) uint4 ring[];   // [DEPTH][NP][NS][threads]
  __shared__ float sm[2][64];
  __shared__ double red[SRC == Src::Mix ? 32 * 4 : 1];
  __shared__ uint4 exchange[DROP && V == 1 ? 1024 : 1];
  pdl_prologue();
  constexpr int NS = SRC == Src::Mix ? 5 : 4;   // Mix: dy, H[0..3]; Add: dy, x, residual, dsum
  const int sub = m.rpc == 1 ? 0 : threadIdx.x / m.tpr, t = threadIdx.x - sub * m.tpr;
  const Packs<V, NP> pk(t, m);
  const int64_t D = a.D;
  const int stride = pk.step * V;
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16u, pitch = blockDim.x * 16u;
  DropSeed seed{};
  DropCol dcol[V > 1 ? NP : 1];
  if constexpr (DROP) drop_cols<V, NP>(seed = drop_seed(a.drop), pk, t, dcol);
  float w[NP][V], dw[NP][V];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
#pragma unroll
    for (int e = 0; e < V; ++e) dw[k][e] = w[k][e] = 0.f;
    if (pk.first + k * pk.step < m.DV) load_w_pack<T, V>(a.weight, a.w_f32, pk.first * V + k * stride, w[k]);
  }

  // where the CTA is: rows base .. base + rpc - 1 of the item, the item's end (32 bits: at most 2^31 - 1 rows, and the
  // counts are unsigned, so that stepping past the last one does not wrap)
  const uint32_t items = (uint32_t)a.items, chunks = (uint32_t)a.chunks, S = (uint32_t)a.S;
  struct Pos { uint32_t item, base, end; };
  auto enter = [&](Pos& q) {   // first rows of q.item
    if (q.item >= items) return;
    if constexpr (SRC == Src::Mix) {
      const uint32_t b = q.item / chunks, c = q.item - b * chunks;
      q.base = b * S + c * m.rpc;
      q.end = (b + 1) * S;
    } else {
      q.base = q.item * m.rpc;
      q.end = min(q.base + m.rpc, S);
    }
  };
  auto next = [&](Pos q) -> Pos {
    q.base += SRC == Src::Mix ? chunks * m.rpc : m.rpc;
    if (SRC == Src::Add || q.base >= q.end) {
      q.item += gridDim.x;
      enter(q);
    }
    return q;
  };
  bool own[NP];   // the packs that exist
#pragma unroll
  for (int k = 0; k < NP; ++k) own[k] = pk.first + k * pk.step < m.DV;
  auto issue = [&](int stage, const Pos& q) -> float {   // starts the copies of a row; its rstd
    const int64_t row = (int64_t)q.base + sub;
    float rstd = 0.f;
    if (q.item < items && row < q.end) {
      rstd = __ldg(a.rstd + row);
      if constexpr (DEPTH == 0) return rstd;
      const T* src[NS];
      src[0] = (const T*)a.dy + row * D + pk.first * V;
      if constexpr (SRC == Src::Mix) {
#pragma unroll
        for (int n = 0; n < 4; ++n) src[1 + n] = (const T*)a.x + (row * 4 + n) * D + pk.first * V;
      } else {
        src[1] = (const T*)a.x + row * D + pk.first * V;
        src[2] = (const T*)a.res + row * D + pk.first * V;
        src[3] = (const T*)a.dsum + row * D + pk.first * V;
      }
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (own[k]) {
#pragma unroll
          for (int n = 0; n < NS; ++n)
            if (SRC == Src::Mix || n < 2 || (n == 2 ? a.res : a.dsum))
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + (uint32_t)((stage * NP + k) * NS + n) * pitch),
                           "l"(src[n] + k * stride)
                           : "memory");
        }
    }
    if constexpr (DEPTH > 0) asm volatile("cp.async.commit_group;" ::: "memory");
    return rstd;
  };
  auto slot = [&](int stage, int k, int n) -> RawPack<T, V> {
    RawPack<T, V> r;
    if constexpr (DEPTH > 0)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.w.x), "=r"(r.w.y), "=r"(r.w.z), "=r"(r.w.w)
                   : "r"(mine + (uint32_t)((stage * NP + k) * NS + n) * pitch)
                   : "memory");
    return r;
  };

  float pre[4] = {0.f, 0.f, 0.f, 0.f};
  double dpre[4] = {0.0, 0.0, 0.0, 0.0};
  uint32_t pre_of = 0xffffffffu;
  int parity = 0, stage = 0;
  float ahead[DEPTH > 1 ? DEPTH - 1 : 1];   // rstd of the rows on the way
  Pos q{blockIdx.x, 0, 0};
  enter(q);
  Pos qi = q;
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) {
    ahead[d] = issue(d, qi);
    qi = next(qi);
  }
  while (q.item < items) {
    float rstd;
    if constexpr (DEPTH <= 1) {
      rstd = issue(0, q);
      if (DEPTH == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
      rstd = ahead[0];
#pragma unroll
      for (int d = 0; d + 1 < DEPTH - 1; ++d) ahead[d] = ahead[d + 1];
      ahead[DEPTH - 2] = issue(stage == 0 ? DEPTH - 1 : stage - 1, qi);   // the stage read in the previous iteration
      qi = next(qi);
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH > 0 ? DEPTH - 1 : 0) : "memory");
    }
    const int64_t row = (int64_t)q.base + sub;
    const bool live = row < q.end;
    const Pos q2 = next(q);
    RawPack<T, V> now[DEPTH == 0 ? NP : 1][NS];
    if constexpr (DEPTH == 0) {   // all at once and without a branch: what does not exist reads the first column of a row that does
      const int64_t r = live ? row : (int64_t)q.base;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int64_t at = own[k] ? pk.first + k * pk.step : 0;
        now[k][0] = ld_raw<T, V>((const T*)a.dy + r * D + at);
        if constexpr (SRC == Src::Mix) {
#pragma unroll
          for (int n = 0; n < 4; ++n) now[k][1 + n] = ld_raw<T, V>((const T*)a.x + (r * 4 + n) * D + at);
        } else {
          now[k][1] = ld_raw<T, V>((const T*)a.x + r * D + at);
        }
      }
      if constexpr (SRC == Src::Add) {
        if (a.res) {
#pragma unroll
          for (int k = 0; k < NP; ++k) now[k][2] = ld_raw<T, V>((const T*)a.res + r * D + (own[k] ? pk.first + k * pk.step : 0));
        }
        if (a.dsum) {
#pragma unroll
          for (int k = 0; k < NP; ++k) now[k][3] = ld_raw<T, V>((const T*)a.dsum + r * D + (own[k] ? pk.first + k * pk.step : 0));
        }
      }
    }
    auto pack = [&](int k, int n) -> RawPack<T, V> {
      if constexpr (DEPTH == 0) return now[k][n];
      else return slot(stage, k, n);
    };
    DropBits<V> bits[DROP ? NP : 1];
    if constexpr (DROP) drop_row_bits<V, NP>(seed, dcol, drop_row(a.drop, seed, row), pk, exchange, bits);
    if constexpr (SRC == Src::Mix) {
      if (q.item != pre_of) {
        pre_of = q.item;
#pragma unroll
        for (int n = 0; n < 4; ++n) pre[n] = __ldg(a.hpre + (int64_t)(q.item / chunks) * 4 + n);
      }
    }
    float s[NP][V], h[NP][V], unused = 0.f;
    Sum2 c2{0};
#pragma unroll
    for (int k = 0; k < NP; ++k) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[k][e] = h[k][e] = 0.f;
      // single elements: selected below; a branch here held their loads back (457 -> 271 us at 16384 x 4095 fp32)
      constexpr bool kSelect = DEPTH == 0 && !DROP;
      if (kSelect || (live && own[k])) {
        const RawPack<T, V> dy = pack(k, 0);
        if constexpr (SRC == Src::Mix) {
          RawPack<T, V> x[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) x[n] = pack(k, 1 + n);
          mix_pack<T, V>(x, pre, s[k]);
        } else {
          unpack<T, V>(pack(k, 1), s[k]);
          if constexpr (DROP) drop_apply<V>(a.drop, bits[k], s[k]);
          if (a.res) {
            float u[V];
            unpack<T, V>(pack(k, 2), u);
            pack_add<V>(s[k], u);
          }
        }
        unpack<T, V>(dy, h[k]);
        pack_scale<V>(h[k], rstd);
        if (kSelect && !(live && own[k])) {
#pragma unroll
          for (int e = 0; e < V; ++e) h[k][e] = s[k][e] = 0.f;
        }
        pack_fma<V>(dw[k], h[k], s[k]);
        pack_mul<V>(h[k], w[k]);
        pack_dot<V>(c2, h[k], s[k]);
      }
    }
    float c = total(c2);
    row_sum_max<false>(c, unused, sm[parity], m, sub);
    parity ^= 1;   // the next row's sums go to the other half: nobody can still be reading it
    const float kk = c * rstd * rstd * a.inv_D;   // c holds one rstd already
    Sum2 acc[4] = {};
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      if (live && own[k]) {
        float g[V];
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = -kk;
        pack_mul_add<V>(g, s[k], h[k]);
        if constexpr (SRC == Src::Mix) {
          T* o = (T*)a.dx + row * 4 * D + pk.first * V + k * stride;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            float x[V], u[V];
            unpack<T, V>(pack(k, 1 + n), x);
            pack_dot<V>(acc[n], g, x);
#pragma unroll
            for (int e = 0; e < V; ++e) u[e] = g[e];
            pack_scale<V>(u, pre[n]);
            PackIO<T, V>::store(o + n * D, u);
          }
        } else {
          if (a.dsum) {
            float u[V];
            unpack<T, V>(pack(k, 3), u);
            pack_add<V>(g, u);
          }
          if constexpr (DROP) {
            if (a.dres) PackIO<T, V>::store((T*)a.dres + row * D + pk.first * V + k * stride, g);
            drop_apply<V>(a.drop, bits[k], g);
          }
          PackIO<T, V>::store((T*)a.dx + row * D + pk.first * V + k * stride, g);
        }
      }
    }
    if constexpr (SRC == Src::Mix) {
#pragma unroll
      for (int n = 0; n < 4; ++n) dpre[n] += (double)total(acc[n]);
      if (q2.item != q.item) {
        __syncthreads();   // the previous item's readers of red are done
        block_store_f64(dpre, a.dpre_part + (int64_t)q.item * 4, red);
#pragma unroll
        for (int n = 0; n < 4; ++n) dpre[n] = 0.0;
      }
    }
    q = q2;
    stage = stage + 1 >= DEPTH ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (a.dw_part) {
    float* o = a.dw_part + ((int64_t)blockIdx.x * m.rpc + sub) * D + pk.first * V;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      if (pk.first + k * pk.step < m.DV) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          if constexpr (V == 1) o[k * stride] = dw[k][0];
          else *reinterpret_cast<float4*>(o + k * stride + e) = make_float4(dw[k][e], dw[k][e + 1], dw[k][e + 2], dw[k][e + 3]);
        }
      }
    }
  }
}

// Ends the backward in 3 us (296 partial rows of 4096), both sums in fp64 and a fixed order.  CTAs [0, wide): out[d] =
// sum_i part[i, d], 32 columns per CTA, 32 threads per column that take rows i, i + 32, ...  CTA wide + b: dH_pre[b] from
// its chunks' four sums.
template <typename T>
__global__ void __launch_bounds__(1024)
k_norm_finish(const float* __restrict__ part, int n, int64_t D, T* __restrict__ out, int wide,
              const float* __restrict__ pre_part, int64_t chunks, float* __restrict__ dpre) {
  pdl_prologue();
  __shared__ double sm[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  double s = 0.0;
  if ((int)blockIdx.x < wide) {
    const int64_t d = (int64_t)blockIdx.x * 32 + c;
    if (d < D) {
      const float* p = part + (int64_t)g * D + d;
      for (int i = g; i < n; i += 32 * 4, p += 32 * 4 * D) {   // four loads in flight
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = i + 32 * u < n ? __ldg(p + (int64_t)32 * u * D) : 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) s += (double)v[u];
      }
    }
    sm[g][c] = s;
    __syncthreads();
    s = warp_sum_f64(sm[c][g]);            // warp g adds the 32 sums of column g
    const int64_t col = (int64_t)blockIdx.x * 32 + g;
    if (c == 0 && col < D) out[col] = from_f32<T>((float)s);
  } else {
    const int64_t b = (int64_t)blockIdx.x - wide;
    const float* p = pre_part + b * chunks * 4;
    for (int64_t i = threadIdx.x; i < chunks * 4; i += 1024) s += (double)__ldg(p + i);   // thread i: sum i % 4
#pragma unroll
    for (int o = 16; o >= 4; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (c < 4) sm[g][c] = s;
    __syncthreads();
    if (g < 4) {
      s = warp_sum_f64(sm[c][g]);
      if (c == 0) dpre[b * 4 + g] = (float)s;
    }
  }
}

// --------------------------------------------------------------------------------------------------- host side
// The backward's persistent grid: two CTAs of 256 threads per SM (its registers allow no more), one of the wider ones.
// Every row a CTA walks abreast leaves one row of dweight partial sums.
static int64_t bwd_ctas(int64_t items, int threads) {
  const int64_t most = (threads > 256 ? 1 : 2) * (int64_t)sm_count();
  return items < most ? items : most;
}
// Shares that the stream-norm backward divides a batch element's tokens into: as many as fill the device's CTAs once (so any
// number of batch elements fills them evenly), but four rounds of rpc tokens each at least, since a share ends with a
// reduction.  A function of the sequence and the width only: a batch element sums in the same order in any batch.
static int64_t mix_chunks(int64_t S, int rpc) {
  const int64_t groups = (S + rpc - 1) / rpc, most = 2 * (int64_t)sm_count(), few = (groups + 3) / 4;
  return groups <= 4 ? (groups > 0 ? 1 : 0) : few < most ? few : most;
}

// Rows per CTA from which the persistent forward is taken: at 4 the two forms take the same time (1184 x 7168: 15 us,
// 2368 x 4096: 16 us, either way), below it the one-shot form is up to half a microsecond faster, and at 4736 x 7168
// the persistent one takes 44 us against 55.
constexpr int kRingRows = 4;
// Shared memory of an SM that the resident CTAs' rings may use together (each has a few hundred bytes of its own beside).
constexpr size_t kRingBytes = 224 * 1024;

// launch_k for a kernel whose dynamic shared memory may exceed the 48 KiB, static included, it gets without asking.
template <auto Kernel, typename... Args>
static void launch_ring(unsigned grid, unsigned block, size_t smem, cudaStream_t st, Args&&... args) {
  static std::atomic<uint32_t> asked{0};   // devices on which the attribute is set
  int dev = 0;
  if (smem > 40 * 1024 && cudaGetDevice(&dev) == cudaSuccess && (dev > 31 || !(asked.load() >> dev & 1))) {
    (void)cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes);
    if (dev < 32) asked.fetch_or(1u << dev);
  }
  launch_k(Kernel, grid, block, smem, st, std::forward<Args>(args)...);
}

// Threads and rows per CTA for rows of D elements in packs of V: `np` packs per thread.
static RowMap row_map(int64_t D, int V, int np) {
  RowMap m;
  m.DV = (int)(D / V);
  m.tpr = V > 1 ? ((m.DV + np - 1) / np + 31) / 32 * 32 : (m.DV + 32 * np - 1) / (32 * np) * 32;
  m.rpc = m.tpr <= 128 ? 256 / m.tpr : 1;
  return m;
}
// Packs per thread of the register kernels: 2 up to 1024 packs per row, 4 up to 2048; 8 single elements up to 8192;
// 0: the row does not fit.
static int packs_per_thread(int64_t D, int V) {
  if (V == 1) return D <= 8192 ? 8 : 0;
  return D / V <= 1024 ? 2 : D / V <= 2048 ? 4 : 0;
}

// Scratch: at most two rows' worth of partial sums per SM and row walked abreast (rpc <= 8, and then D <= 512), plus the
// chunks' dH_pre sums.
static int64_t dw_rows(int64_t D) { return 2 * (int64_t)sm_count() * (D <= 512 ? 8 : D <= 1024 ? 4 : D <= 2048 ? 2 : 1); }
int64_t rms_norm_bwd_scratch_bytes(int64_t rows, int64_t D) {
  const int64_t n = dw_rows(D);
  return ((rows < n ? (rows + 7) / 8 * 8 : n) * D + 4) * (int64_t)sizeof(float);
}
int64_t stream_norm_bwd_scratch_bytes(int64_t B, int64_t S, int64_t D) {
  return (dw_rows(D) * D + B * mix_chunks(S, 1) * 4 + 4) * (int64_t)sizeof(float);
}

// Arguments common to all entry points of this file.
static int check_norm(const char* what, int64_t rows, int64_t D, int dtype, const void* weight, int wdtype) {
  if (int e = check_bsd_pub(what, 1, 0, D, dtype)) return e;
  if (rows < 0 || rows > kMaxGridItems) return fail(MHC_ERR_BAD_SHAPE, "%s: rows %lld out of range", what, (long long)rows);
  if (weight && wdtype != MHC_F32 && wdtype != dtype)
    return fail(MHC_ERR_BAD_DTYPE, "%s: the weight must be fp32 or of the activation type", what);
  return MHC_OK;
}

static int check_quant(const char* what, int64_t group, int scale_type) {
  if (group != 0 && group != 32 && group != 64 && group != 128)
    return fail(MHC_ERR_BAD_ARGUMENT, "%s: group %lld is not 0 (row), 32, 64 or 128", what, (long long)group);
  if (scale_type != MHC_SCALE_F32 && scale_type != MHC_SCALE_E8M0)
    return fail(MHC_ERR_BAD_ARGUMENT, "%s: unknown scale type %d", what, scale_type);
  return MHC_OK;
}

static void set_scales(NormFwd& a, void* scales, int64_t group, int scale_type, int64_t D) {
  a.scales = scales;
  a.group = (int)group;
  a.shift = group == 32 ? 5 : group == 64 ? 6 : 7;
  a.G = group ? (int)((D + group - 1) / group) : 1;
  a.e8m0 = scale_type == MHC_SCALE_E8M0;
  a.scales8 = a.e8m0 && group == 32 && a.G % 8 == 0 && is_aligned_to(a.scales, 8);
}

static void set_inv(NormFwd& a, int64_t D) {
  const double inv = 1.0 / (double)D;
  a.inv_D = (float)inv;
  a.inv_D_lo = (float)(inv - (double)a.inv_D);
}

template <Src SRC, bool DROP, Out OUT>
static int launch_fwd(const char* what, const NormFwd& a, int dtype, cudaStream_t st) {
  ProfScope ps(SRC == Src::Mix ? "k_stream_norm_fwd" : "k_rms_norm_fwd", st);
  const int vec = pick_vec(dtype, a.D, {a.x, a.res, a.weight, a.sum_out, a.y});
  const int np = packs_per_thread(a.D, vec);
  if (np == 0) {
    MHC_TYPE_DISPATCH(dtype, (launch_k(k_norm_any_fwd<T, SRC, DROP, OUT>, (unsigned)a.rows, 256, 0, st, a)));
    return check_launch(what);
  }
  const RowMap m = row_map(a.D, vec, np);
  const unsigned grid = (unsigned)((a.rows + m.rpc - 1) / m.rpc), block = (unsigned)(m.tpr * m.rpc);
  const size_t smem = (size_t)2 * block * np * (SRC == Src::Mix ? 4 : 2) * 16;
  const int per_sm = std::min(1024 / (int)block, (int)(kRingBytes / smem));
  if ((DROP || OUT != Out::Plain) && np == 2 && per_sm > 0 && grid >= (unsigned)(kRingRows * per_sm * sm_count())) {
    MHC_TYPE_DISPATCH(dtype, (launch_ring<k_norm_fwd_ring<T, vec_width<T>::value, 2, SRC, DROP, OUT>>((unsigned)(per_sm * sm_count()),
                                          block, smem, st, a, m)));
    return check_launch(what);
  }
  if (vec == 1) MHC_TYPE_DISPATCH(dtype, (launch_k(k_norm_fwd<T, 1, 8, SRC, DROP, OUT>, grid, block, 0, st, a, m)));
  else if (np == 2) MHC_TYPE_DISPATCH(dtype, (launch_k(k_norm_fwd<T, vec_width<T>::value, 2, SRC, DROP, OUT>, grid, block, 0, st, a, m)));
  else MHC_TYPE_DISPATCH(dtype, (launch_k(k_norm_fwd<T, vec_width<T>::value, 4, SRC, DROP, OUT>, grid, block, 0, st, a, m)));
  return check_launch(what);
}

// Fills in what depends on the kernel chosen (items, chunks, partial rows) and launches; a.items are rows (Add) or
// batch elements (Mix) on entry.
template <Src SRC, bool DROP>
static int launch_bwd(const char* what, NormBwd& a, float* scratch, int dtype, cudaStream_t st) {
  ProfScope ps(SRC == Src::Mix ? "k_stream_norm_bwd" : "k_rms_norm_bwd", st);
  const int vec = pick_vec(dtype, a.D, {a.dy, a.dsum, a.x, a.res, a.weight, a.dx, a.dres});
  const int np = packs_per_thread(a.D, vec);
  RowMap m{256, 1, 0};
  if (np) m = row_map(a.D, vec, np);
  if constexpr (SRC == Src::Mix) {
    a.chunks = mix_chunks(a.S, m.rpc);
    a.items *= a.chunks;
  } else {
    a.S = a.items;
    a.items = (a.S + m.rpc - 1) / m.rpc;
  }
  const int threads = m.tpr * m.rpc;
  const int64_t ctas = bwd_ctas(a.items, threads);
  a.parts = (int)(ctas * m.rpc);
  scratch = (float*)(((uintptr_t)scratch + 15) & ~(uintptr_t)15);
  if (a.dw_part) { a.dw_part = scratch; scratch += a.parts * a.D; }
  a.dpre_part = scratch;
  const size_t stage = (size_t)threads * np * (SRC == Src::Mix ? 5 : 4) * 16;
  if (np == 0)
    MHC_TYPE_DISPATCH(dtype, (launch_k(k_norm_any_bwd<T, SRC, DROP>, (unsigned)ctas, 256, 0, st, a)));
  else if (vec == 1 && threads <= 512)
    MHC_TYPE_DISPATCH(dtype, (launch_k(k_norm_bwd<T, 1, 8, 0, 512, SRC, DROP>, (unsigned)ctas, threads, 0, st, a, m)));
  else if (vec == 1)
    MHC_TYPE_DISPATCH(dtype, (launch_k(k_norm_bwd<T, 1, 8, 0, 1024, SRC, DROP>, (unsigned)ctas, threads, 0, st, a, m)));
  else if (np == 4)
    MHC_TYPE_DISPATCH(dtype, (launch_ring<k_norm_bwd<T, vec_width<T>::value, 4, 1, 512, SRC, DROP>>((unsigned)ctas, threads, stage, st, a, m)));
  else   // three stages: 229 instead of 207 us at 32768 x 4096 bf16
    MHC_TYPE_DISPATCH(dtype, (launch_ring<k_norm_bwd<T, vec_width<T>::value, 2, 2, 512, SRC, DROP>>((unsigned)ctas, threads, 2 * stage, st, a, m)));
  return check_launch(what);
}

// dweight (null: none) from the CTAs' partial rows, dH_pre (Mix; null: none) from the chunks' sums.
static int finish_bwd(const char* what, const NormBwd& a, void* dweight, int wdtype, float* dpre, int64_t B, cudaStream_t st) {
  if (!dweight && !dpre) return MHC_OK;
  const int wide = dweight ? (int)((a.D + 31) / 32) : 0;
  const int64_t grid = wide + (dpre ? B : 0);
  if (grid > kMaxGridItems) return fail(MHC_ERR_BAD_SHAPE, "%s: too many batch elements", what);
  ProfScope ps("k_norm_finish", st);
  MHC_TYPE_DISPATCH(wdtype, (launch_k(k_norm_finish<T>, (unsigned)grid, 1024, 0, st, (const float*)a.dw_part, a.parts, a.D,
                                      (T*)dweight, wide, (const float*)a.dpre_part, a.chunks, dpre)));
  return check_launch(what);
}

int stream_norm_fwd_impl(const void* H, const float* H_pre, const void* weight, int wdtype, void* bi, void* y,
                         float* rstd, int64_t B, int64_t S, int64_t D, int dtype, float eps, cudaStream_t st) {
  NormFwd a{};
  a.x = H; a.hpre = H_pre; a.weight = weight; a.w_f32 = wdtype == MHC_F32; a.sum_out = bi; a.y = y; a.rstd = rstd;
  a.rows = B * S; a.S = S; a.D = D; a.eps = eps; set_inv(a, D);
  return launch_fwd<Src::Mix, false, Out::Plain>("stream_norm_fwd", a, dtype, st);
}

}  // namespace mhc

using namespace mhc;

extern "C" int mhc_add_rms_norm_fwd(const void* x, const void* residual, const void* weight, int weight_dtype,
                                    const int64_t* rng, int drop_threshold, int64_t row_offset, void* sum_out, void* y,
                                    float* rstd, int64_t rows, int64_t D, int dtype, float eps, mhc_stream_t stream) {
  const char* what = "add_rms_norm_fwd";
  if (int e = check_norm(what, rows, D, dtype, weight, weight_dtype)) return e;
  if (!(eps >= 0.f)) return fail(MHC_ERR_BAD_ARGUMENT, "%s: eps must not be negative", what);
  NormFwd a{};
  const bool drop = drop_threshold != 0;
  if (drop)
    if (int e = make_drop(what, rng, drop_threshold, row_offset, rows, &a.drop)) return e;
  if (rows == 0 || D == 0) return MHC_OK;
  if (!x || !y) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
  a.x = x; a.res = residual; a.weight = weight; a.w_f32 = weight_dtype == MHC_F32; a.sum_out = sum_out; a.y = y;
  a.rstd = rstd; a.rows = rows; a.S = 1; a.D = D; a.eps = eps; set_inv(a, D);
  cudaStream_t st = (cudaStream_t)stream;
  return drop ? launch_fwd<Src::Add, true, Out::Plain>(what, a, dtype, st)
              : launch_fwd<Src::Add, false, Out::Plain>(what, a, dtype, st);
}

extern "C" int mhc_add_rms_norm_quant_fwd(const void* x, const void* residual, const void* weight, int weight_dtype,
                                          void* sum_out, void* q, void* scales, int64_t group, int scale_type,
                                          int64_t rows, int64_t D, int dtype, float eps, mhc_stream_t stream) {
  const char* what = "add_rms_norm_quant_fwd";
  if (int e = check_norm(what, rows, D, dtype, weight, weight_dtype)) return e;
  if (int e = check_quant(what, group, scale_type)) return e;
  if (!(eps >= 0.f)) return fail(MHC_ERR_BAD_ARGUMENT, "%s: eps must not be negative", what);
  if (rows == 0 || D == 0) return MHC_OK;
  if (!x || !q || !scales) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
  NormFwd a{};
  a.x = x; a.res = residual; a.weight = weight; a.w_f32 = weight_dtype == MHC_F32; a.sum_out = sum_out; a.y = q;
  set_scales(a, scales, group, scale_type, D);
  a.rows = rows; a.S = 1; a.D = D; a.eps = eps; set_inv(a, D);
  cudaStream_t st = (cudaStream_t)stream;
  return group ? launch_fwd<Src::Add, false, Out::GroupScale>(what, a, dtype, st)
               : launch_fwd<Src::Add, false, Out::RowScale>(what, a, dtype, st);
}

extern "C" int mhc_rms_norm_bwd(const void* dy, const void* dsum, const void* x, const void* residual, const float* rstd,
                                const void* weight, int weight_dtype, const int64_t* rng, int drop_threshold, int64_t row_offset, void* dx,
                                void* dresidual, void* dweight, void* scratch, int64_t scratch_bytes, int64_t rows,
                                int64_t D, int dtype, mhc_stream_t stream) {
  const char* what = "rms_norm_bwd";
  if (int e = check_norm(what, rows, D, dtype, weight, weight_dtype)) return e;
  NormBwd a{};
  const bool drop = drop_threshold != 0;
  if (drop)
    if (int e = make_drop(what, rng, drop_threshold, row_offset, rows, &a.drop)) return e;
  if (D == 0) return MHC_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (dweight && weight_dtype != MHC_F32 && weight_dtype != dtype)
    return fail(MHC_ERR_BAD_DTYPE, "%s: the weight must be fp32 or of the activation type", what);
  if (rows == 0) {
    if (dweight && cudaMemsetAsync(dweight, 0, D * (weight_dtype == MHC_F32 ? 4 : 2), st) != cudaSuccess) return check_launch(what);
    return MHC_OK;
  }
  if (dweight && scratch_bytes < rms_norm_bwd_scratch_bytes(rows, D))
    return fail(MHC_ERR_SCRATCH_TOO_SMALL, "%s: scratch %lld < %lld bytes", what, (long long)scratch_bytes,
                (long long)rms_norm_bwd_scratch_bytes(rows, D));
  if (!dy || !x || !rstd || !dx || (dweight && !scratch)) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
  if (!is_aligned_to(scratch, 4)) return fail(MHC_ERR_MISALIGNED, "%s: scratch must be 4-byte aligned", what);
  if (!drop && dresidual) return fail(MHC_ERR_BAD_ARGUMENT, "%s: without dropout the residual's gradient is dx", what);
  a.dy = dy; a.dsum = dsum; a.x = x; a.res = residual; a.rstd = rstd; a.weight = weight; a.w_f32 = weight_dtype == MHC_F32;
  a.dx = dx; a.dres = dresidual; a.dw_part = dweight ? (float*)scratch : nullptr; a.items = rows; a.D = D; a.inv_D = (float)(1.0 / (double)D);
  if (int e = drop ? launch_bwd<Src::Add, true>(what, a, (float*)scratch, dtype, st)
                   : launch_bwd<Src::Add, false>(what, a, (float*)scratch, dtype, st))
    return e;
  return finish_bwd(what, a, dweight, weight_dtype, nullptr, 0, st);
}

extern "C" int mhc_stream_norm_fwd(const void* H, const float* H_pre, const void* weight, int weight_dtype,
                                   void* branch_input, void* y, float* rstd, int64_t B, int64_t S, int64_t D, int dtype,
                                   float eps, mhc_stream_t stream) {
  const char* what = "stream_norm_fwd";
  if (int e = check_bsd_pub(what, B, S, D, dtype)) return e;
  if (int e = check_norm(what, rows_of(B, S), D, dtype, weight, weight_dtype)) return e;
  if (!(eps >= 0.f)) return fail(MHC_ERR_BAD_ARGUMENT, "%s: eps must not be negative", what);
  if (B == 0 || S == 0 || D == 0) return MHC_OK;
  if (!H || !H_pre || !y) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
  return stream_norm_fwd_impl(H, H_pre, weight, weight_dtype, branch_input, y, rstd, B, S, D, dtype, eps,
                              (cudaStream_t)stream);
}

extern "C" int mhc_stream_norm_quant_fwd(const void* H, const float* H_pre, const void* weight, int weight_dtype,
                                         void* q, void* scales, int64_t group, int scale_type, int64_t B, int64_t S,
                                         int64_t D, int dtype, float eps, mhc_stream_t stream) {
  const char* what = "stream_norm_quant_fwd";
  if (int e = check_bsd_pub(what, B, S, D, dtype)) return e;
  if (int e = check_norm(what, rows_of(B, S), D, dtype, weight, weight_dtype)) return e;
  if (int e = check_quant(what, group, scale_type)) return e;
  if (!(eps >= 0.f)) return fail(MHC_ERR_BAD_ARGUMENT, "%s: eps must not be negative", what);
  if (B == 0 || S == 0 || D == 0) return MHC_OK;
  if (!H || !H_pre || !q || !scales) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
  NormFwd a{};
  a.x = H; a.hpre = H_pre; a.weight = weight; a.w_f32 = weight_dtype == MHC_F32; a.y = q;
  set_scales(a, scales, group, scale_type, D); a.rows = B * S; a.S = S; a.D = D; a.eps = eps; set_inv(a, D);
  cudaStream_t st = (cudaStream_t)stream;
  return group ? launch_fwd<Src::Mix, false, Out::GroupScale>(what, a, dtype, st)
               : launch_fwd<Src::Mix, false, Out::RowScale>(what, a, dtype, st);
}

extern "C" int mhc_stream_norm_bwd(const void* dy, const void* H, const float* H_pre, const float* rstd,
                                   const void* weight, int weight_dtype, void* dH, float* dH_pre, void* dweight,
                                   void* scratch, int64_t scratch_bytes, int64_t B, int64_t S, int64_t D, int dtype,
                                   mhc_stream_t stream) {
  const char* what = "stream_norm_bwd";
  if (int e = check_bsd_pub(what, B, S, D, dtype)) return e;
  if (int e = check_norm(what, rows_of(B, S), D, dtype, weight, weight_dtype)) return e;
  if (dweight && weight_dtype != MHC_F32 && weight_dtype != dtype)
    return fail(MHC_ERR_BAD_DTYPE, "%s: the weight must be fp32 or of the activation type", what);
  cudaStream_t st = (cudaStream_t)stream;
  if (B == 0 || S == 0 || D == 0) {
    if (B > 0 && !dH_pre) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
    if ((B > 0 && cudaMemsetAsync(dH_pre, 0, B * 4 * sizeof(float), st) != cudaSuccess) ||
        (dweight && D > 0 && cudaMemsetAsync(dweight, 0, D * (weight_dtype == MHC_F32 ? 4 : 2), st) != cudaSuccess))
      return check_launch(what);
    return MHC_OK;
  }
  if (scratch_bytes < stream_norm_bwd_scratch_bytes(B, S, D))
    return fail(MHC_ERR_SCRATCH_TOO_SMALL, "%s: scratch %lld < %lld bytes", what, (long long)scratch_bytes,
                (long long)stream_norm_bwd_scratch_bytes(B, S, D));
  if (!dy || !H || !H_pre || !rstd || !dH || !dH_pre || !scratch) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
  if (!is_aligned_to(scratch, 4)) return fail(MHC_ERR_MISALIGNED, "%s: scratch must be 4-byte aligned", what);
  NormBwd a{};
  a.dy = dy; a.x = H; a.hpre = H_pre; a.rstd = rstd; a.weight = weight; a.w_f32 = weight_dtype == MHC_F32; a.dx = dH;
  a.dw_part = dweight ? (float*)scratch : nullptr; a.items = B; a.S = S; a.D = D;
  a.inv_D = (float)(1.0 / (double)D);
  if (int e = launch_bwd<Src::Mix, false>(what, a, (float*)scratch, dtype, st)) return e;
  return finish_bwd(what, a, dweight, weight_dtype, dH_pre, B, st);
}
