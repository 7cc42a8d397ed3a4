// Dropout with counter-based masks (rng.cuh): y = x * keep / (1 - p).  The backward is the same map applied to
// the upstream gradient.
#include "common.cuh"
#include "launch.h"
#include "rng.cuh"

namespace mhc {

// A thread owns one group of columns (a 16-byte pack; for V = 1, rows that do not divide into packs, 8 columns read one
// by one) and walks kDropRows rows: the column's part of the generator is computed once and all loads are
// issued before the first use.
#ifndef MHC_DROPOUT_MINB
#define MHC_DROPOUT_MINB 6
#endif
#ifndef MHC_DROP_ROWS
#define MHC_DROP_ROWS 4
#endif
constexpr int kDropRows = MHC_DROP_ROWS;
struct DropGeo {
  int64_t rows, D;
  int groups;   // column groups of a row
  int cols;     // column groups per CTA (threads abreast in a row)
  int sub;      // rows abreast
  int CG;       // CTAs side by side in a row
};

template <typename T, int V>
__global__ void __launch_bounds__(256, MHC_DROPOUT_MINB)
k_counter_dropout(const T* __restrict__ x, T* __restrict__ y, DropGeo g, Drop drop) {
  pdl_prologue();
  const int64_t chunk = g.CG == 1 ? blockIdx.x : blockIdx.x / g.CG;
  const int cg = g.CG == 1 ? 0 : (int)(blockIdx.x - chunk * g.CG);
  const int s = threadIdx.x / g.cols, pos = cg * g.cols + threadIdx.x - s * g.cols;
  const DropSeed seed = drop_seed(drop);   // whole warps
  if (pos >= g.groups) return;
  const int64_t row0 = chunk * (kDropRows * g.sub) + s, step = g.sub;
  if constexpr (V > 1) {
    const uint32_t col = (uint32_t)pos * V;
    const int64_t left = g.rows - row0, jump = step * g.D;
    const int n = left <= 0 ? 0 : left > (kDropRows - 1) * step ? kDropRows : (int)((left + step - 1) / step);   // rows to do
    const T* xp = x + row0 * g.D + col;
    T* yp = y + row0 * g.D + col;
    RawPack<T, V> raw[kDropRows];
#pragma unroll
    for (int r = 0; r < kDropRows; ++r)
      if (r < n) raw[r] = ld_raw<T, V>(xp + r * jump);
    const DropCol dc = drop_col(seed, col >> 3);
#pragma unroll
    for (int r = 0; r < kDropRows; ++r) {
      if (r < n) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = raw_get<V>(raw[r], e);
        drop_apply<V>(drop, drop_bits<V>(seed, dc, drop_row(drop, seed, row0 + r * step), col), v);
        PackIO<T, V>::store(yp + r * jump, v);
      }
    }
  } else {
    const int64_t col = (int64_t)pos * 8;
    const DropCol dc = drop_col(seed, (uint32_t)pos);
#pragma unroll
    for (int r = 0; r < kDropRows; ++r) {
      const int64_t row = row0 + r * step, base = row * g.D + col;
      if (row < g.rows) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = col + e < g.D ? to_f32(x[base + e]) : 0.f;
        drop_apply<8>(drop, drop_bits<8>(seed, dc, drop_row(drop, seed, row), col), v);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < g.D) y[base + e] = from_f32<T>(v[e]);
      }
    }
  }
}

int make_drop(const char* what, const int64_t* rng, int threshold, int64_t row_offset, int64_t rows, Drop* out) {
  if (threshold < 1 || threshold > 65535)
    return fail(MHC_ERR_BAD_ARGUMENT, "%s: drop threshold %d is not in 1..65535", what, threshold);
  if (row_offset < 0 || rows < 0 || row_offset > (1LL << 32) - rows)
    return fail(MHC_ERR_BAD_ARGUMENT, "%s: rows %lld from offset %lld exceed 2^32", what, (long long)rows, (long long)row_offset);
  if (!rng) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer (rng)", what);
  if (!is_aligned_to(rng, 8)) return fail(MHC_ERR_MISALIGNED, "%s: rng must be 8-byte aligned", what);
  out->rng = rng;
  out->thr = (uint32_t)threshold;
  out->scale = (float)(65536.0 / (65536.0 - (double)threshold));
  out->row0 = (uint32_t)row_offset;
  return MHC_OK;
}

}  // namespace mhc

using namespace mhc;

extern "C" int mhc_counter_dropout(const void* x, const int64_t* rng, int drop_threshold, int64_t row_offset, void* y,
                                   int64_t rows, int64_t D, int dtype, mhc_stream_t stream) {
  const char* what = "counter_dropout";
  if (int e = check_bsd_pub(what, 1, 0, D, dtype)) return e;
  if (rows < 0 || rows > (1LL << 32)) return fail(MHC_ERR_BAD_SHAPE, "%s: rows %lld out of range", what, (long long)rows);
  Drop drop;
  if (int e = make_drop(what, rng, drop_threshold, row_offset, rows, &drop)) return e;
  if (rows == 0 || D == 0) return MHC_OK;
  if (!x || !y) return fail(MHC_ERR_NULL_POINTER, "%s: null pointer", what);
  const int vec = pick_vec(dtype, D, {x, y});
  DropGeo g;
  g.rows = rows;
  g.D = D;
  g.groups = (int)(vec > 1 ? D / vec : (D + 7) / 8);
  g.cols = g.groups >= 256 ? 256 : (g.groups + 31) / 32 * 32;
  g.sub = 256 / g.cols;
  g.CG = (g.groups + g.cols - 1) / g.cols;
  const int64_t grid = (rows + kDropRows * g.sub - 1) / (kDropRows * g.sub) * g.CG;
  if (grid > kMaxGridItems) return fail(MHC_ERR_BAD_SHAPE, "%s: too many work items (%lld)", what, (long long)grid);
  cudaStream_t st = (cudaStream_t)stream;
  {
    ProfScope ps("k_counter_dropout", st);
    MHC_DISPATCH(dtype, vec, (launch_k(k_counter_dropout<T, V>, (unsigned)grid, (unsigned)(g.cols * g.sub), 0, st,
                                       (const T*)x, (T*)y, g, drop)));
  }
  return check_launch(what);
}
