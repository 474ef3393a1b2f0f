// Per-row 8-bit quantisation (lf_quantize_rows): a token's activations, or an output
// channel's weights, as whole multiples of the row's largest magnitude / 127 (the
// formula and its rounding: lf_quant.cuh).
//
// The bound is HBM: each element is read once and one byte is written.  So a row stays
// in registers between the search for its largest magnitude and the rounding: 1, 2, 4 or
// 8 warps share a row (8 to 32 elements a lane, rows up to 8,192), 16-byte loads, all of a
// row's loads in flight before the first is used; six CTAs of 8 warps an SM.  Longer rows
// are read a second time (from L2).  Rows that are not 16-byte aligned or whose length is
// not a multiple of 8 are read in pairs at 16 bits, one element a load at 32 (or where q's
// rows are not 8-byte aligned).
// Measured, bf16: 17,410 rows of 4,096 36.8 us (5.8 TB/s), of 1,024 14.3 us with launch;
// 16,384 of 10,240, read twice, 100 us (5.0 TB/s counted once); 17,410 of 4,095 58 us (72 with
// one element a load).
#include "lf_common.cuh"
#include "lf_internal.h"
#include "lf_quant.cuh"

namespace lf {

namespace {

constexpr int kThreads = 256;
// Column numbers are 32-bit, and a chunk past the row's end is formed before it is found empty:
// 8 warps' chunks of 256, and a lane's eight columns.
constexpr int kMaxCols = INT32_MAX - 4096;

struct QuantParams {
  const void* x;
  int64_t ldx, n_rows;
  int32_t cols;
  int8_t* q;
  int64_t ldq;
  float* scale;
};

// WPR warps per row, each with kChunks chunks of 256 elements in registers; LONG: rows of
// any length, the rest read twice.
// VEC: 8 neighbours a lane, read as one (NEAR: 16-bit rows of any alignment, as pairs).
template <typename T, int WPR, int kChunks, bool VEC, bool NEAR, bool LONG>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && VEC && !LONG ? 6 : 1) quantize_rows_kernel(const QuantParams p) {
  __shared__ uint32_t s_top[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = warp % WPR;
  const int64_t row = int64_t(blockIdx.x) * (kThreads / 32 / WPR) + warp / WPR;
  const bool live = row < p.n_rows;
  pdl_wait();
  pdl_launch_dependents();
  const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.ldx;
  int8_t* q = p.q + (live ? row : 0) * p.ldq;
  auto load = [&](QuantChunk<T, VEC>& c, int32_t base) {
    if constexpr (NEAR) c.load_near(x, base, lane, p.cols);
    else c.load(x, base, lane, p.cols);
  };
  QuantChunk<T, VEC> v[kChunks];
  uint32_t top = 0;
  if (live) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) load(v[c], (c * WPR + sub) * 256);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) top = sizeof(T) == 2 ? __vmaxu2(top, v[c].top()) : max(top, v[c].top());
    if constexpr (LONG) {
      for (int32_t base = (kChunks * WPR + sub) * 256; base < p.cols; base += WPR * 256) {
        QuantChunk<T, VEC> w;
        load(w, base);
        top = sizeof(T) == 2 ? __vmaxu2(top, w.top()) : max(top, w.top());
      }
    }
  }
  if constexpr (sizeof(T) == 2) top = max(top >> 16, top & 0xffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (WPR > 1) {
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = max(top, s_top[warp - sub + i]);
  }
  if (!live) return;
  const RowQuant rq(top_bits<T>(top));
  if (sub == 0 && lane == 0) p.scale[row] = rq.scale;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) v[c].store(q, (c * WPR + sub) * 256, lane, p.cols, rq);
  if constexpr (LONG) {
    for (int32_t base = (kChunks * WPR + sub) * 256; base < p.cols; base += WPR * 256) {
      QuantChunk<T, VEC> w;
      load(w, base);
      w.store(q, base, lane, p.cols, rq);
    }
  }
}

template <typename T, int WPR, int kChunks, bool LONG>
int launch_rows(const QuantParams& p, bool vec, bool near, cudaStream_t s) {
  constexpr int rows = kThreads / 32 / WPR;
  const int64_t blocks = (p.n_rows + rows - 1) / rows;
  if (blocks > INT32_MAX) return set_error(LF_ERR_UNSUPPORTED, "lf_quantize_rows: %lld rows", (long long)p.n_rows);
  constexpr bool kNear = sizeof(T) == 2;
  const cudaError_t e = launch_pdl(vec             ? quantize_rows_kernel<T, WPR, kChunks, true, false, LONG>
                                   : kNear && near ? quantize_rows_kernel<T, WPR, kChunks, kNear, kNear, LONG>
                                                   : quantize_rows_kernel<T, WPR, kChunks, false, false, LONG>,
                                   dim3(unsigned(blocks)), dim3(kThreads), 0, s, p);
  if (e != cudaSuccess) return cuda_error(e, "launch quantize_rows");
  count_launch();
  return LF_OK;
}

// A row's 256-element chunks over 1, 2, 4 or 8 warps, three or four a warp (so that a row of
// 2,560 leaves 2 of 12 empty, not 6 of 16).
template <typename T>
int launch_quantize(const QuantParams& p, bool vec, bool near, cudaStream_t s) {
  const int n = (p.cols + 255) / 256;
  if (n <= 1) return launch_rows<T, 1, 1, false>(p, vec, near, s);
  if (n <= 2) return launch_rows<T, 1, 2, false>(p, vec, near, s);
  if (n <= 3) return launch_rows<T, 1, 3, false>(p, vec, near, s);
  if (n <= 4) return launch_rows<T, 1, 4, false>(p, vec, near, s);
  if (n <= 6) return launch_rows<T, 2, 3, false>(p, vec, near, s);
  if (n <= 8) return launch_rows<T, 2, 4, false>(p, vec, near, s);
  if (n <= 12) return launch_rows<T, 4, 3, false>(p, vec, near, s);
  if (n <= 16) return launch_rows<T, 4, 4, false>(p, vec, near, s);
  if (n <= 24) return launch_rows<T, 8, 3, false>(p, vec, near, s);
  if (n <= 32) return launch_rows<T, 8, 4, false>(p, vec, near, s);
  return launch_rows<T, 8, 4, true>(p, vec, near, s);
}

}  // namespace

}  // namespace lf

using namespace lf;

extern "C" int lf_quantize_rows(void* stream, int dtype, const void* x, int64_t ldx, int64_t n_rows, int cols,
                                int8_t* q, int64_t ldq, float* scale) {
  if (dtype != LF_DTYPE_BF16 && dtype != LF_DTYPE_F16 && dtype != LF_DTYPE_F32)
    return set_error(LF_ERR_INVALID, "lf_quantize_rows: unknown dtype %d", dtype);
  if (n_rows < 0 || cols <= 0) return set_error(LF_ERR_INVALID, "lf_quantize_rows: %lld rows of %d", (long long)n_rows, cols);
  if (cols > kMaxCols)
    return set_error(LF_ERR_UNSUPPORTED, "lf_quantize_rows: rows of %d above %d elements", cols, kMaxCols);
  if (n_rows == 0) return LF_OK;
  if (x == nullptr || q == nullptr || scale == nullptr)
    return set_error(LF_ERR_INVALID, "lf_quantize_rows: null x, q or scale");
  if (ldx < cols || ldq < cols) return set_error(LF_ERR_INVALID, "lf_quantize_rows: a row stride is below %d", cols);
  const int es = dtype == LF_DTYPE_F32 ? 4 : 2;
  QuantParams p{x, ldx, n_rows, cols, q, ldq, scale};
  const bool near = (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0;
  const bool vec = near && cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (ldx * es) % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == LF_DTYPE_BF16) return launch_quantize<__nv_bfloat16>(p, vec, near, s);
  if (dtype == LF_DTYPE_F16) return launch_quantize<__half>(p, vec, near, s);
  return launch_quantize<float>(p, vec, near, s);
}
