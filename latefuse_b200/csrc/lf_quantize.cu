// Per-row 8-bit quantisation (lf_quantize_rows): a token's activations, or an output
// channel's weights, as whole multiples of the row's largest magnitude / 127 (the
// formula and its rounding: lf_quant.cuh).
//
// The bound is HBM: each element is read once and one byte is written.  So a row stays
// in registers between the search for its largest magnitude and the rounding: 1, 2, 4 or
// 8 warps share a row (32 elements a lane, rows up to 8,192), 16-byte loads, all of a
// row's loads in flight before the first is used.  Longer rows are read a second time
// (from L2), and rows that are not 16-byte aligned or whose length is not a multiple of
// 8 take one element per load, 32 neighbours to a warp.
#include "lf_common.cuh"
#include "lf_internal.h"
#include "lf_quant.cuh"

namespace lf {

namespace {

constexpr int kThreads = 256;
constexpr int kChunks = 4;  // 8 elements each, per lane

struct QuantParams {
  const void* x;
  int64_t ldx, n_rows;
  int32_t cols;
  int8_t* q;
  int64_t ldq;
  float* scale;
};

// This lane's 8 elements of chunk c: neighbours (VEC), or 32 apart.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int32_t base, int lane, int32_t cols, float (&v)[8]) {
  if constexpr (VEC) {
    const int32_t col = base + lane * 8;
    if (col < cols) {
      if constexpr (sizeof(T) == 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + col);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Pack2<T>::unpack(u[i]);
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      } else {
        const float4 a = *reinterpret_cast<const float4*>(row + col), b = *reinterpret_cast<const float4*>(row + col + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int32_t col = base + i * 32 + lane;
      v[i] = col < cols ? DT<T>::to_f(row[col]) : 0.f;
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(int8_t* row, int32_t base, int lane, int32_t cols, const RowQuant& rq,
                                       const float (&v)[8]) {
  if constexpr (VEC) {
    const int32_t col = base + lane * 8;
    if (col < cols) {
      uint2 w;
      w.x = rq.q4(v[0], v[1], v[2], v[3]);
      w.y = rq.q4(v[4], v[5], v[6], v[7]);
      *reinterpret_cast<uint2*>(row + col) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int32_t col = base + i * 32 + lane;
      if (col < cols) row[col] = int8_t(rq.q(v[i]));
    }
  }
}

// WPR warps per row; rows of at most WPR * 1024 elements, or any length when LONG (WPR = 8).
template <typename T, int WPR, bool VEC, bool LONG>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantParams p) {
  __shared__ uint32_t s_top[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = warp % WPR;
  const int64_t row = int64_t(blockIdx.x) * (kThreads / 32 / WPR) + warp / WPR;
  const bool live = row < p.n_rows;
  pdl_wait();
  pdl_launch_dependents();
  const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.ldx;
  int8_t* q = p.q + (live ? row : 0) * p.ldq;
  float v[kChunks][8];
  uint32_t top = 0;
  if (live) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) load8<T, VEC>(x, (c * WPR + sub) * 256, lane, p.cols, v[c]);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, mag_bits(v[c][i]));
    if constexpr (LONG) {
      for (int32_t base = (kChunks * WPR + sub) * 256; base < p.cols; base += WPR * 256) {
        float w[8];
        load8<T, VEC>(x, base, lane, p.cols, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, mag_bits(w[i]));
      }
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (WPR > 1) {
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = max(top, s_top[warp - sub + i]);
  }
  if (!live) return;
  const RowQuant rq(top);
  if (sub == 0 && lane == 0) p.scale[row] = rq.scale;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) store8<VEC>(q, (c * WPR + sub) * 256, lane, p.cols, rq, v[c]);
  if constexpr (LONG) {
    for (int32_t base = (kChunks * WPR + sub) * 256; base < p.cols; base += WPR * 256) {
      float w[8];
      load8<T, VEC>(x, base, lane, p.cols, w);
      store8<VEC>(q, base, lane, p.cols, rq, w);
    }
  }
}

template <typename T>
int launch_quantize(const QuantParams& p, bool vec, cudaStream_t s) {
  const int wpr = p.cols <= 1024 ? 1 : p.cols <= 2048 ? 2 : p.cols <= 4096 ? 4 : 8;
  const int rows = kThreads / 32 / wpr;
  const int64_t blocks = (p.n_rows + rows - 1) / rows;
  if (blocks > INT32_MAX) return set_error(LF_ERR_UNSUPPORTED, "lf_quantize_rows: %lld rows", (long long)p.n_rows);
  const bool lng = p.cols > 8192;
  auto kern = wpr == 1   ? (vec ? quantize_rows_kernel<T, 1, true, false> : quantize_rows_kernel<T, 1, false, false>)
              : wpr == 2 ? (vec ? quantize_rows_kernel<T, 2, true, false> : quantize_rows_kernel<T, 2, false, false>)
              : wpr == 4 ? (vec ? quantize_rows_kernel<T, 4, true, false> : quantize_rows_kernel<T, 4, false, false>)
              : lng      ? (vec ? quantize_rows_kernel<T, 8, true, true> : quantize_rows_kernel<T, 8, false, true>)
                         : (vec ? quantize_rows_kernel<T, 8, true, false> : quantize_rows_kernel<T, 8, false, false>);
  const cudaError_t e = launch_pdl(kern, dim3(unsigned(blocks)), dim3(kThreads), 0, s, p);
  if (e != cudaSuccess) return cuda_error(e, "launch quantize_rows");
  count_launch();
  return LF_OK;
}

}  // namespace

}  // namespace lf

using namespace lf;

extern "C" int lf_quantize_rows(void* stream, int dtype, const void* x, int64_t ldx, int64_t n_rows, int cols,
                                int8_t* q, int64_t ldq, float* scale) {
  if (dtype != LF_DTYPE_BF16 && dtype != LF_DTYPE_F16 && dtype != LF_DTYPE_F32)
    return set_error(LF_ERR_INVALID, "lf_quantize_rows: unknown dtype %d", dtype);
  if (n_rows < 0 || cols <= 0) return set_error(LF_ERR_INVALID, "lf_quantize_rows: %lld rows of %d", (long long)n_rows, cols);
  if (n_rows == 0) return LF_OK;
  if (x == nullptr || q == nullptr || scale == nullptr)
    return set_error(LF_ERR_INVALID, "lf_quantize_rows: null x, q or scale");
  if (ldx < cols || ldq < cols) return set_error(LF_ERR_INVALID, "lf_quantize_rows: a row stride is below %d", cols);
  const int es = dtype == LF_DTYPE_F32 ? 4 : 2;
  QuantParams p{x, ldx, n_rows, cols, q, ldq, scale};
  const bool vec = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (ldx * es) % 16 == 0 &&
                   (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == LF_DTYPE_BF16) return launch_quantize<__nv_bfloat16>(p, vec, s);
  if (dtype == LF_DTYPE_F16) return launch_quantize<__half>(p, vec, s);
  return launch_quantize<float>(p, vec, s);
}
