// Dropout with counter-based masks (rng.cuh): y = x * keep / (1 - p).  The backward is the same map applied to
// the upstream gradient.
#include "common.cuh"
#include "launch.h"
#include "rng.cuh"

namespace mhc {

// A thread owns one 16-byte pack of columns and walks kDropRows rows: the column's part of the generator is computed once
// and all loads are issued before the first use.  Bound by the generator's instructions (ALU pipe 58 %, 2.9 of 4 issue
// slots): 92 us at 32768 x 4096 bf16, 5.8 TB/s.  4 or 6 rows take 96, 5 or 7 CTAs per SM 102 or 99, a shared-memory ring
// over 8 to 32 rows 105 to 120.  fp32, where two threads compute the same block for four columns each: 48 us at 8192 x 4096
// (41 at the memory's rate), 90 at 8192 x 8192 (82).
#ifndef MHC_DROPOUT_MINB
#define MHC_DROPOUT_MINB 6
#endif
#ifndef MHC_DROP_ROWS
#define MHC_DROP_ROWS 5
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
}

// Rows that do not divide into packs: a warp owns 256 columns of kDropRows rows.  A lane computes the block of one group of
// 8 columns, the warp exchanges the halves through shared memory of its own, and every access is to consecutive elements.
template <typename T>
__global__ void __launch_bounds__(256)
k_counter_dropout_scalar(const T* __restrict__ x, T* __restrict__ y, DropGeo g, Drop drop) {
  __shared__ uint4 exchange[8][32];
  pdl_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 8 + warp, chunk = id / g.CG;
  const int col0 = (int)(id - chunk * g.CG) * 256;
  const DropSeed seed = drop_seed(drop);
  const DropCol dc = drop_col(seed, (uint32_t)(col0 >> 3) + lane);
  for (int64_t row = chunk * kDropRows; row < min((chunk + 1) * kDropRows, g.rows); ++row) {   // uniform over the warp
    const T* xp = x + row * g.D + col0 + lane;
    T* yp = y + row * g.D + col0 + lane;
    RawPack<T, 1> raw[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col0 + k * 32 + lane < g.D) raw[k] = ld_raw<T, 1>(xp + k * 32);
    __syncwarp();
    exchange[warp][lane] = drop_block(seed, dc, drop_row(drop, seed, row));
    __syncwarp();
    const uint16_t* h = reinterpret_cast<const uint16_t*>(exchange[warp]) + lane;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col0 + k * 32 + lane < g.D) {
        DropBits<1> b;
        b.w[0] = (uint32_t)h[k * 32] << 16;
        float v[1] = {raw_get<1>(raw[k], 0)};
        drop_apply<1>(drop, b, v);
        yp[k * 32] = from_f32<T>(v[0]);
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
  if (vec == 1) {
    g.CG = (int)((D + 255) / 256);
    const int64_t grid = ((rows + kDropRows - 1) / kDropRows * g.CG + 7) / 8;
    if (grid > kMaxGridItems) return fail(MHC_ERR_BAD_SHAPE, "%s: too many work items (%lld)", what, (long long)grid);
    ProfScope ps("k_counter_dropout", (cudaStream_t)stream);
    MHC_TYPE_DISPATCH(dtype, (launch_k(k_counter_dropout_scalar<T>, (unsigned)grid, 256, 0, (cudaStream_t)stream, (const T*)x,
                                       (T*)y, g, drop)));
    return check_launch(what);
  }
  g.groups = (int)(D / vec);
  g.cols = g.groups >= 256 ? 256 : (g.groups + 31) / 32 * 32;
  g.sub = 256 / g.cols;
  g.CG = (g.groups + g.cols - 1) / g.cols;
  const int64_t grid = (rows + kDropRows * g.sub - 1) / (kDropRows * g.sub) * g.CG;
  if (grid > kMaxGridItems) return fail(MHC_ERR_BAD_SHAPE, "%s: too many work items (%lld)", what, (long long)grid);
  cudaStream_t st = (cudaStream_t)stream;
  {
    ProfScope ps("k_counter_dropout", st);
    MHC_TYPE_DISPATCH(dtype, (launch_k(k_counter_dropout<T, vec_width<T>::value>, (unsigned)grid, (unsigned)(g.cols * g.sub), 0, st,
                                       (const T*)x, (T*)y, g, drop)));
  }
  return check_launch(what);
}
