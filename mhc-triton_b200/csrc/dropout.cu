// Dropout with counter-based masks (rng.cuh): y = x * keep / (1 - p).  The backward is the same map applied to
// the upstream gradient.
#include "common.cuh"
#include "launch.h"
#include "rng.cuh"

namespace mhc {

// One thread per pack of V columns (V > 1), or per group of 8 columns read one by one (V = 1: rows that do not
// divide into 16-byte packs).
template <typename T, int V>
__global__ void __launch_bounds__(256)
k_counter_dropout(const T* __restrict__ x, T* __restrict__ y, int64_t items, uint32_t per_row, int64_t D, Drop drop) {
  pdl_prologue();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= items) return;
  const DropKey key = drop_key(drop);
  const int64_t row = i <= 0xffffffffLL ? (int64_t)((uint32_t)i / per_row) : i / per_row;
  const int64_t pos = i - row * per_row;
  if constexpr (V > 1) {
    float v[V];
    const int64_t col = pos * V;
    PackIO<T, V>::load(x + row * D + col, v);
    drop_apply<V>(drop, drop_bits<V>(drop, key, row, col), v);
    PackIO<T, V>::store(y + row * D + col, v);
  } else {
    const int64_t col = pos * 8, base = row * D + col;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = col + e < D ? to_f32(x[base + e]) : 0.f;
    drop_apply<8>(drop, drop_bits<8>(drop, key, row, col), v);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < D) y[base + e] = from_f32<T>(v[e]);
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
  const int64_t per_row = vec > 1 ? D / vec : (D + 7) / 8, items = rows * per_row, grid = (items + 255) / 256;
  if (grid > kMaxGridItems) return fail(MHC_ERR_BAD_SHAPE, "%s: too many work items (%lld)", what, (long long)grid);
  cudaStream_t st = (cudaStream_t)stream;
  {
    ProfScope ps("k_counter_dropout", st);
    MHC_DISPATCH(dtype, vec, (launch_k(k_counter_dropout<T, V>, (unsigned)grid, 256, 0, st, (const T*)x, (T*)y, items,
                                       (uint32_t)per_row, D, drop)));
  }
  return check_launch(what);
}
