// Projection in 8-bit integers on tcgen05 (kind::i8): for int8 x (m, k) with a scale per
// row (token) and int8 w (n, k) with a scale per row (output channel),
//     y = act(float(sum_k x w) * x_scale * w_scale + bias)
// The sum is exact in 32-bit integers (127^2 k < 2^31 up to k = 133,144; calls stop at
// 131,072), so the result does not depend on tile, split or order; it becomes f32 (one
// rounding), is scaled and biased in f32 (the scale of w and the bias in one FMA), and
// the activation's result is rounded once to the output type.
//
// Two kernels, the same results bit for bit:
//
// linear_int8_kernel, for batches: the bf16 projection's CTA-pair GEMM (lf_linear.cu) with
// 8-bit operands.  256 x 256 output tiles on persistent clusters of two CTAs, K blocks of
// 128 (128 bytes: the same SW128 boxes, ring and barriers), tcgen05.mma.cta_group::2
// M = 256, N = 256, K = 32.  A K block has the bytes of bf16's 64-wide one and twice its
// multiplications in the same time.
//   warp 0      TMA producer (both CTAs): an x box {128, 128} and a w box {128, 128} into
//               a 6-stage ring, completing on the leader's barrier;
//   warp 1      MMA issuer (leader only); TMEM holds two 256-column accumulators;
//   warps 2-17  epilogue (both CTAs), four warps per TMEM lane quadrant, 64 columns each,
//               32 at a time: staged per warp and written by TMA, or by the warp row by row
//               where y's rows are not 16-byte aligned.
//
// linear_int8_split_kernel, for few tokens, where streaming w is the bound and 256-wide
// tiles would leave most SMs without work: w's rows are the MMA's M (128 channels per
// CTA), the tokens its N (16 to 128), and K is split over a cluster of up to 8 CTAs whose
// integer partial sums meet in distributed shared memory (each CTA finishes a share of
// the tokens).  Integer addition is exact, so the split changes no bit.  Up to 16 float rows
// of up to 4,096 are quantised in the same launch, by the warps that finish later on: a
// launch of their own takes the host 2 us and a workspace.
//
// Every wait is bounded: a timeout sets LF_STATUS_TIMEOUT and the roles unwind.
#include <cstring>

#include "lf_common.cuh"
#include "lf_internal.h"
#include "lf_pair.cuh"
#include "lf_quant.cuh"

namespace lf {

namespace {

constexpr int kBK = 128;  // K block: 128 int8 = one SW128 row

struct alignas(64) LinearInt8Params {
  CUtensorMap x_map;  // 2D {K, M} uint8, box {128, rows}, SW128
  CUtensorMap w_map;  // 2D {K, N} uint8, box {128, 128}, SW128
  CUtensorMap y_map;  // 2D {N, M}, box {32, 32}: SW64 for 2-byte y, SW128 for f32 (tma_out)
  const float* x_scale;
  const float* w_scale;
  const void* bias;   // N entries or null
  void* y;
  int64_t ldy;
  int64_t m_rows;
  int32_t n, n_tiles, n_tiles_n, n_kb;
  int32_t tma_out;    // y's base and row stride are 16-byte aligned
  int32_t vec_ch;     // w_scale and bias are aligned for pairs
  int32_t split;      // split kernel: CTAs of the cluster that share a tile's K
  const void* rows;   // float rows, quantised on chip (m_rows <= kRowsM), or null
  int64_t ld_rows;
  int32_t k;
  int32_t vec_rows;   // they are aligned for 8 elements a load
  int32_t* status;
};

// D[tmem] (+)= A * B, 8-bit integers into s32.
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor for kind::i8: signed 8-bit A and B, both K-major, s32 D.
__host__ __device__ constexpr uint32_t umma_idesc_i8(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ bool aborted(const int32_t* f) { return *reinterpret_cast<const volatile int32_t*>(f) != 0; }

// The GELU of two values for a 16-bit result, v max(0, sign v) - |v| Phi(-|v|) with
//     Phi(-z) = exp(-z^2 / 2) R(z),  R(z) = erfcx(z / sqrt 2) / 2,
// R as a polynomial in min(z, 5) - 5/2 whose largest relative error is least: degree 11 for
// bf16 (2^-18.8 of R), degree 12 for f16 (2^-20.7).  With the roundings of its evaluation
// (2^-19.7 at most) and of the exponent (2^-19) |v| Phi(-|v|) is within 2^-17.4 (bf16) and
// 2^-17.9 (f16) of its value, within 2^-18.4 and 2^-19.6 for |v| up to 2; beyond 5, where R is
// held, it is below 1.5e-6, still falls with the exponential and is within 3.7%.  So
// results are the formula's but where it lies next to a border between two 16-bit values:
// 0.016% of normal inputs round the other way in bf16 and 0.033% in f16, where the formula
// in f32 has 0.002% and 0.014% (degrees 8 and 10 had 0.9% and 0.5%).
// One SFU operation a value where gelu2_fast takes two: with K = 1024 the epilogue's GELU
// sets the projection's time (17,410 x 4,096, bf16 and f16: 76 and 77 us; 67 and 73 with
// degrees 8 and 10, 54 without an activation).
template <typename T>
__device__ __forceinline__ float2 gelu2_narrow(float2 v) {
  constexpr bool kBf16 = DT<T>::umma_fmt == 1;
  constexpr int kDegree = kBf16 ? 11 : 12;
  constexpr float kR[2][13] = {
      {1.1876396754928464e-08f, -6.810693520264977e-08f, 1.1003712074852956e-07f, -3.798999443915818e-07f,
       3.342534455441637e-06f, -1.5777091903146356e-05f, 6.238623609533533e-05f, -0.0002551310753915459f,
       0.0010172546608373523f, -0.0038328650407493114f, 0.0136485006660223f, -0.04561358690261841f,
       0.14133130013942719f},
      {-5.840812988822108e-08f, 3.262648817781155e-07f, -5.428102554105863e-07f, 1.8756209101411514e-06f,
       -1.4787478903599549e-05f, 6.693375325994566e-05f, -0.0002577411360107362f, 0.0010109581053256989f,
       -0.003830085974186659f, 0.013651634566485882f, -0.04561440274119377f, 0.14133106172084808f}};
  const float2 z = make_float2(fminf(fabsf(v.x), 5.f), fminf(fabsf(v.y), 5.f));
  const float2 l = f2_mul(f2_mul(v, f2(-0.72134752044448170f)), v);  // -v^2 / 2 to base 2
  const float2 u = f2_add(z, f2(-2.5f));
  float2 r = f2(kR[kBf16][0]);
#pragma unroll
  for (int i = 1; i <= kDegree; ++i) r = f2_fma(r, u, f2(kR[kBf16][i]));
  const float2 h = f2_mul(r, make_float2(-sfu_ex2(l.x), -sfu_ex2(l.y)));
  return f2_fma(z, h, make_float2(fmaxf(v.x, 0.f), fmaxf(v.y, 0.f)));
}

// Two accumulators: scaled, biased, activated (f32).
template <typename T, int kAct>
__device__ __forceinline__ float2 finish2(int a0, int a1, float2 xs, float2 ws, float2 b) {
  const float2 y = f2_fma(f2_mul(make_float2(__int2float_rn(a0), __int2float_rn(a1)), xs), ws, b);
  if constexpr (kAct == LF_ACT_GELU) {
    if constexpr (sizeof(T) == 2) return gelu2_narrow<T>(y);
    else return gelu2_fast(y);
  }
  return y;
}

// 32 rows x 32 columns of TMEM in the layout of an mma accumulator: lane 4 r + q holds, of
// the 8-column group j, columns 8 j + 2 q and the next, of rows r and r + 8 (v[4 j .. 4 j + 3])
// and of rows r + 16 and r + 24 (v[16 + 4 j ..]).  A lane then needs the scales of 8 columns
// instead of 32: the epilogue's reads of scales from L1 were competing with the MMAs'
// operand reads.
__device__ __forceinline__ void tmem_ld_frag32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr), "r"(taddr + (16u << 16))
      : "memory");
}

// ---------------------------------------------------------------------------
// batches: CTA pairs, 256 x 256 tiles
// ---------------------------------------------------------------------------
constexpr int kBM = 128, kBN = 256;
constexpr int kABytes = kBM * kBK;         // 16 KB: this CTA's x rows
constexpr int kBBytes = (kBN / 2) * kBK;   // 16 KB: this CTA's half of the w rows
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kEpiWarps = 16;               // a multiple of 4: kEpiWarps / 4 warps per TMEM lane quadrant
constexpr int kWarpCols = kBN / (kEpiWarps / 4);  // columns of the tile per epilogue warp
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kOutCols = 32;
__host__ __device__ constexpr int out_buf(int es) { return 32 * kOutCols * es; }  // one 32 x 32 staging tile
// ring stages: what the staging tiles leave of the shared memory
__host__ __device__ constexpr int stages(int es) {
  const int n = (232448 - 2048 - kEpiWarps * out_buf(es)) / kStageBytes;
  return n < 6 ? n : 6;
}
constexpr int smem_bytes(int es) { return 1024 + stages(es) * kStageBytes + kEpiWarps * out_buf(es) + 1024; }
static_assert(smem_bytes(4) <= 232448 && smem_bytes(2) <= 232448, "above the 227 KB of shared memory a CTA may use");

// A lane's columns of a 32-column chunk (8 j + 2 fq and the next): their scales and biases,
// the biases as they lie in memory, 0 past n.  Loaded a chunk ahead of their use.
template <typename T>
struct Channels {
  float2 ws[4];
  T b[4][2];
  __device__ __forceinline__ void load(const float* w_scale, const T* bias, int32_t col, int32_t n, bool vec) {
    if (vec && col + 25 < n) {  // every pair exists and is aligned as a pair
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ws[j] = __ldg(reinterpret_cast<const float2*>(w_scale + col + 8 * j));
        if (bias != nullptr) {
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint32_t*>(b[j]) = __ldg(reinterpret_cast<const uint32_t*>(bias + col + 8 * j));
          else
            *reinterpret_cast<float2*>(b[j]) = __ldg(reinterpret_cast<const float2*>(bias + col + 8 * j));
        } else {
          b[j][0] = b[j][1] = DT<T>::from_f(0.f);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t c = col + 8 * j;
        ws[j] = make_float2(c < n ? __ldg(w_scale + c) : 0.f, c + 1 < n ? __ldg(w_scale + c + 1) : 0.f);
        b[j][0] = bias != nullptr && c < n ? bias[c] : DT<T>::from_f(0.f);
        b[j][1] = bias != nullptr && c + 1 < n ? bias[c + 1] : DT<T>::from_f(0.f);
      }
    }
  }
  __device__ __forceinline__ float2 bias_of(int j) const { return make_float2(DT<T>::to_f(b[j][0]), DT<T>::to_f(b[j][1])); }
};

// A CTA pair's walk over the output tiles, every n_pairs-th in row-block order, without a
// division a step.
struct TileWalk {
  int32_t t, rb, c;       // tile, row block, column tile
  int32_t n_tiles, n_cols, step, step_rb, step_c;
  __device__ __forceinline__ TileWalk(const LinearInt8Params& p, int pair, int n_pairs) {
    t = pair;
    n_tiles = p.n_tiles;
    n_cols = p.n_tiles_n;
    step = n_pairs;
    rb = pair / n_cols;
    c = pair % n_cols;
    step_rb = n_pairs / n_cols;
    step_c = n_pairs % n_cols;
  }
  __device__ __forceinline__ bool live() const { return t < n_tiles; }
  __device__ __forceinline__ void next() {
    t += step;
    rb += step_rb;
    c += step_c;
    if (c >= n_cols) {
      c -= n_cols;
      ++rb;
    }
  }
};

// A staged 32 x 32 block into rows that are not 16-byte aligned, eight rows of 32 columns in
// flight (17,410 x 1,024 -> 4,095: 117 us one row at a time, 72 so; with GELU 131 and 103, now 111).
// Out of line: inlined it took registers from the aligned epilogue (GELU 71 -> 74 us then).
template <typename T>
__device__ __noinline__ void store_rows(const uint8_t* block, T* dst, int64_t ld, int64_t rows, int32_t cols, int lane) {
  constexpr int kRowBytes = kOutCols * sizeof(T);
  const int left = rows < 32 ? int(rows) : 32, live = lane < cols ? left : 0, byte = lane * int(sizeof(T));
  dst += lane;
#pragma unroll 1
  for (int r0 = 0; r0 < left; r0 += 8) {
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rs = sizeof(T) == 2 ? (i >> 1) & 3 : i;
      o[i] = *reinterpret_cast<const T*>(block + (r0 + i) * kRowBytes + (((byte >> 4) ^ rs) << 4) + (byte & 15));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (r0 + i < live) *dst = o[i];
      dst += ld;
    }
  }
}

template <typename T, int kAct>
__global__ void __launch_bounds__(kThreads, 1) linear_int8_kernel(const __grid_constant__ LinearInt8Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const uint32_t rank = uniform(cluster_ctarank());  // 0: the leader, which issues the MMAs
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  constexpr int kOutBuf = out_buf(sizeof(T)), kStages = stages(sizeof(T));

  const uint32_t s_out0 = base + kStages * kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(gbase + kStages * kStageBytes + kEpiWarps * kOutBuf);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  constexpr int FULL = 0, EMPTY = kStages, ACC_FULL = 2 * kStages, ACC_EMPTY = ACC_FULL + 2, DRAIN = ACC_EMPTY + 2,
                N_BARS = DRAIN + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(&bars[N_BARS]);
  int32_t* s_abort = reinterpret_cast<int32_t*>(tmem_slot + 1);

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar(FULL + i), 1);   // the leader's arrive, with both CTAs' bytes
      mbar_init(bar(EMPTY + i), 1);  // the leader's MMA commit
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ACC_FULL + i), 1);
      mbar_init(bar(ACC_EMPTY + i), 2 * kEpiWarps);  // both CTAs' epilogue warps
    }
    mbar_init(bar(DRAIN), 1);
    *s_abort = 0;
    fence_mbar_init();
    prefetch_tmap(&p.x_map);
    prefetch_tmap(&p.w_map);
    if (p.tma_out) prefetch_tmap(&p.y_map);  // no map is made of other rows
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc_pair(smem_u32(tmem_slot), 2 * kBN);
  }
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before either signals the other's
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  pdl_wait();
  pdl_launch_dependents();

  auto wait = [&](uint32_t b, uint32_t parity) { return warp_wait(b, parity, s_abort, p.status); };

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    int kk = 0;
    bool stop = false;
    for (TileWalk w(p, pair, n_pairs); w.live() && !stop; w.next()) {
      const int32_t m0 = w.rb * (2 * kBM) + int32_t(rank) * kBM;
      const int32_t n0 = w.c * kBN + int32_t(rank) * (kBN / 2);
      for (int kb = 0; kb < p.n_kb; ++kb, ++kk) {
        const int s = kk % kStages;
        if (!wait(bar(EMPTY + s), ((kk / kStages) & 1) ^ 1)) {
          stop = true;
          break;
        }
        if (elect_one()) {
          const uint32_t st = base + s * kStageBytes;
          const uint32_t full = mapa_shared(bar(FULL + s), 0);
          if (rank == 0) mbar_arrive_expect_tx(bar(FULL + s), 2 * kStageBytes);
          tma_load_2d_pair(st, &p.x_map, full, kb * kBK, m0);
          tma_load_2d_pair(st + kABytes, &p.w_map, full, kb * kBK, n0);
        }
        __syncwarp();
      }
    }
    if (aborted(s_abort) && rank == 0) {  // loads nobody consumed land before the CTA exits (bounded)
      for (int q = (kk > kStages ? kk - kStages : 0); q < kk; ++q)
        mbar_wait(bar(FULL + q % kStages), (q / kStages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (the leader)
    if (rank == 0) {
      constexpr uint32_t idesc = umma_idesc_i8(2 * kBM, kBN);
      const uint64_t a_desc = smem_desc(base, 16, 1024, 2), b_desc = smem_desc(base + kABytes, 16, 1024, 2);
      int kk = 0, n_it = 0;
      bool stop = false;
      for (TileWalk w(p, pair, n_pairs); w.live() && !stop; w.next(), ++n_it) {
        const int a = n_it & 1;
        if (!wait(bar(ACC_EMPTY + a), ((n_it >> 1) & 1) ^ 1)) break;
        tc_fence_after();
        for (int kb = 0; kb < p.n_kb; ++kb, ++kk) {
          const int s = kk % kStages;
          if (!wait(bar(FULL + s), (kk / kStages) & 1)) {
            stop = true;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t off = uint64_t(s * (kStageBytes >> 4));
#pragma unroll
            for (int q = 0; q < kBK / 32; ++q)  // 32 bytes of K a step
              umma_i8_pair(tmem + a * kBN, a_desc + off + uint64_t(2 * q), b_desc + off + uint64_t(2 * q), idesc,
                           (kb | q) != 0 ? 1u : 0u);
            umma_commit_pair(bar(EMPTY + s));
            if (kb == p.n_kb - 1) umma_commit_pair(bar(ACC_FULL + a));
          }
          __syncwarp();
        }
      }
      if (aborted(s_abort)) {  // every issued MMA finishes before TMEM is released (bounded)
        if (elect_one()) umma_commit_pair_local(bar(DRAIN));
        __syncwarp();
        mbar_wait(bar(DRAIN), 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..17, both CTAs)
    const int quad = warp & 3;
    const int c0 = ((warp - 2) >> 2) * kWarpCols;  // this warp's columns of the tile
    const uint32_t taddr = tmem + (uint32_t(quad * 32) << 16) + c0;
    const uint32_t my_out = s_out0 + (warp - 2) * kOutBuf;
    uint8_t* g_out = gbase + (my_out - base);
    const uint32_t acc_empty = mapa_shared(bar(ACC_EMPTY), 0);  // the leader's
    const T* bias = static_cast<const T*>(p.bias);
    T* y = static_cast<T*>(p.y);
    const int fr = lane >> 2, fq = lane & 3;  // this lane's rows fr + 8 k and columns 8 j + 2 fq of a 32 x 32 block
    const bool vec = p.vec_ch != 0;
    // scales and biases come a chunk ahead, the rows' scales a tile ahead
    Channels<T> next;
    float xs_next[4];
    auto col_of = [&](const TileWalk& w) { return w.c * kBN + c0 + 2 * fq; };
    auto row_of = [&](const TileWalk& w) { return int64_t(w.rb) * (2 * kBM) + int64_t(rank) * kBM + quad * 32; };
    auto load_xs = [&](const TileWalk& w) {
      const int64_t m = row_of(w) + fr;
#pragma unroll
      for (int k = 0; k < 4; ++k) xs_next[k] = m + 8 * k < p.m_rows ? __ldg(p.x_scale + m + 8 * k) : 0.f;
    };
    TileWalk w(p, pair, n_pairs);
    if (w.live()) {
      next.load(p.w_scale, bias, col_of(w), p.n, vec);
      load_xs(w);
    }
    for (int n_it = 0; w.live(); ++n_it) {
      const int a = n_it & 1;
      const int64_t m0 = row_of(w);  // this warp's 32 rows
      const int32_t n0 = w.c * kBN + c0;
      float xs[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) xs[k] = xs_next[k];
      w.next();  // from here on the tile after
      if (w.live()) load_xs(w);
      if (!wait(bar(ACC_FULL + a), (n_it >> 1) & 1)) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kWarpCols; c += kOutCols) {
        const int32_t col0 = n0 + c;
        const Channels<T> ch = next;
        if (c + kOutCols < kWarpCols) next.load(p.w_scale, bias, col0 + kOutCols + 2 * fq, p.n, vec);
        else if (w.live()) next.load(p.w_scale, bias, col_of(w), p.n, vec);
        if (col0 >= p.n) continue;
        uint32_t v[32];
        tmem_ld_frag32(taddr + a * kBN + c, v);
        // the store that last read this staging tile must be done with it
        if (lane == 0) tma_store_wait_read_all();
        __syncwarp();
        // rows of 64 bytes: SW64, 16-byte chunk q of row r at q ^ ((r >> 1) & 3); of 128
        // bytes (f32): SW128, at q ^ (r & 7).  fr + 8 k has fr's swizzle.
        constexpr int kRowBytes = kOutCols * sizeof(T);
        const int swz = sizeof(T) == 2 ? (fr >> 1) & 3 : fr & 7;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 cb = ch.bias_of(j);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int i = (k >> 1) * 16 + j * 4 + (k & 1) * 2;
            const float2 r = finish2<T, kAct>(int(v[i]), int(v[i + 1]), f2(xs[k]), ch.ws[j], cb);
            uint8_t* dst = g_out + (fr + 8 * k) * kRowBytes;
            if constexpr (sizeof(T) == 2)
              *reinterpret_cast<uint32_t*>(dst + ((j ^ swz) << 4) + fq * 4) = Pack2<T>::pack(r.x, r.y);
            else
              *reinterpret_cast<float2*>(dst + (((2 * j + (fq >> 1)) ^ swz) << 4) + (fq & 1) * 8) = r;
          }
        }
        if (p.tma_out) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.y_map, my_out, col0, int32_t(m0));
            tma_store_commit();
          }
        } else {  // rows that are not 16-byte aligned: 32 neighbouring columns of a row at a time
          __syncwarp();
          store_rows<T>(g_out, y + m0 * p.ldy + col0, p.ldy, p.m_rows - m0, p.n - col0, lane);
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(acc_empty + a * 8);  // this warp's TMEM reads of the tile are done
    }
    if (lane == 0) tma_store_wait_all();
  }

  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still signal its barriers or read its operands
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem, 2 * kBN);
  }
}

// ---------------------------------------------------------------------------
// few tokens: 128 channels x NT tokens per CTA, K split over a cluster
// ---------------------------------------------------------------------------
constexpr int kSplitEpiWarps = 8;  // two per TMEM lane quadrant
constexpr int kSplitThreads = 64 + 32 * kSplitEpiWarps;
__host__ __device__ constexpr int split_stages(int nt) { return nt <= 32 ? 8 : 6; }
__host__ __device__ constexpr int split_stage_bytes(int nt) { return 128 * kBK + nt * kBK; }
constexpr int split_smem_bytes(int nt) { return 1024 + split_stages(nt) * split_stage_bytes(nt) + 512; }
static_assert(split_smem_bytes(128) <= 232448 && split_smem_bytes(32) <= 232448, "shared memory");
// float rows: up to 16 of 4,096, whose integers (NT x 128 bytes a K block) stay beside the ring
constexpr int kRowsM = 16, kRowsK = 4096;
constexpr int rows_smem_bytes() { return split_smem_bytes(kRowsM) + kRowsM * kRowsK; }
static_assert(rows_smem_bytes() <= 232448, "shared memory");
// the partial sums (NT x 128 int32) reuse the ring
static_assert(128 * 128 * 4 <= 6 * split_stage_bytes(128) && 16 * 128 * 4 <= 8 * split_stage_bytes(16), "ring");

__device__ __forceinline__ int4 ld_dsmem_i4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// kRows, the finishing warps before the product: p.rows' scales, and their integers of this
// CTA's K blocks [kb0, kb1) in the layout that a TMA load of them would have (K-major SW128,
// NT rows a block).  Every CTA finds the rows' largest magnitudes for itself, from L2.
template <typename T, bool VEC>
__device__ __forceinline__ void quantize_share(const LinearInt8Params& p, uint8_t* blocks, uint32_t* s_top, float* s_scale,
                                               int kb0, int kb1, int w, int lane) {
  const int m = int(p.m_rows), share = m <= 1 ? 8 : m <= 2 ? 4 : m <= 4 ? 2 : 1;  // warps a row
  const T* x = static_cast<const T*>(p.rows);
  for (int r = w / share; r < m; r += kSplitEpiWarps / share) {
    uint32_t top = 0;
    for (int32_t base = (w % share) * 256; base < p.k; base += 4 * share * 256) {
      QuantChunk<T, VEC> c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i].load(x + r * p.ld_rows, base + i * share * 256, lane, p.k);
#pragma unroll
      for (int i = 0; i < 4; ++i) top = sizeof(T) == 2 ? __vmaxu2(top, c[i].top()) : max(top, c[i].top());
    }
    if constexpr (sizeof(T) == 2) top = max(top >> 16, top & 0xffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) atomicMax(&s_top[r], top);
  }
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kSplitEpiWarps) : "memory");  // every row's largest magnitude is known
  const int chunks = (kb1 - kb0 + 1) / 2;
  for (int r = w / share; r < m; r += kSplitEpiWarps / share) {
    const RowQuant rq(top_bits<T>(s_top[r]));
    if (lane == 0 && w % share == 0) s_scale[r] = rq.scale;
    uint8_t* row = blocks + (r >> 3) * 1024 + (r & 7) * 128;
    for (int c = w % share; c < chunks; c += share) {
      QuantChunk<T, VEC> v;
      v.load(x + r * p.ld_rows, kb0 * kBK + c * 256, lane, p.k);
      const uint2 q = v.steps(rq);
      if constexpr (VEC) {  // bytes 8 l .. 8 l + 7 of two blocks, 16 lanes a block
        const int kb = 2 * c + (lane >> 4), piece = (lane & 15) >> 1;
        if (kb < kb1 - kb0)
          *reinterpret_cast<uint2*>(row + kb * (kRowsM * kBK) + ((piece ^ (r & 7)) << 4) + (lane & 1) * 8) = q;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = i * 32 + lane, kb = 2 * c + (at >> 7), piece = (at & 127) >> 4;
          if (kb < kb1 - kb0)
            row[kb * (kRowsM * kBK) + ((piece ^ (r & 7)) << 4) + (at & 15)] =
                uint8_t((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xffu);
        }
      }
    }
  }
}

template <typename T, int NT, int kAct, bool kRows>
__global__ void __launch_bounds__(kSplitThreads, 1) linear_int8_split_kernel(const __grid_constant__ LinearInt8Params p) {
  constexpr int kSt = split_stages(NT), kSb = split_stage_bytes(NT);
  constexpr int kLoad = kRows ? 128 * kBK : kSb;  // bytes that arrive in a stage
  constexpr uint32_t kTmemCols = NT < 32 ? 32 : NT;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const int S = p.split;
  const int rank = int(uniform(cluster_ctarank()));
  const int32_t n0 = int32_t(blockIdx.x / unsigned(S)) * 128;
  const int64_t m0 = int64_t(blockIdx.y) * NT;
  const int kb0 = int(int64_t(p.n_kb) * rank / S), kb1 = int(int64_t(p.n_kb) * (rank + 1) / S);

  uint8_t* blocks = gbase + kSt * kSb;  // kRows: the rows' integers
  uint64_t* bars = reinterpret_cast<uint64_t*>(blocks + (kRows ? kRowsM * kRowsK : 0));
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  constexpr int FULL = 0, EMPTY = kSt, ACC = 2 * kSt, ROWS = ACC + 1, N_BARS = ROWS + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(&bars[N_BARS]);
  int32_t* s_abort = reinterpret_cast<int32_t*>(tmem_slot + 1);
  uint32_t* s_top = tmem_slot + 2;
  float* s_scale = reinterpret_cast<float*>(s_top + kRowsM);
  if (tid == 0) {
    for (int i = 0; i < kSt; ++i) {
      mbar_init(bar(FULL + i), 1);
      mbar_init(bar(EMPTY + i), 1);
    }
    mbar_init(bar(ACC), 1);
    mbar_init(bar(ROWS), kSplitEpiWarps);
    *s_abort = 0;
    fence_mbar_init();
    if constexpr (!kRows) prefetch_tmap(&p.x_map);
    prefetch_tmap(&p.w_map);
  }
  if (kRows && warp == 2 && lane < kRowsM) s_top[lane] = 0;
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    int kk = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++kk) {
      const int s = kk % kSt;
      if (!warp_wait(bar(EMPTY + s), ((kk / kSt) & 1) ^ 1, s_abort, p.status)) break;
      if (elect_one()) {
        const uint32_t st = base + s * kSb;
        mbar_arrive_expect_tx(bar(FULL + s), kLoad);
        tma_load_2d(st, &p.w_map, bar(FULL + s), kb * kBK, n0);
        if constexpr (!kRows) tma_load_2d(st + 128 * kBK, &p.x_map, bar(FULL + s), kb * kBK, int32_t(m0));
      }
      __syncwarp();
    }
    if (aborted(s_abort))  // loads nobody consumed land before the CTA exits (bounded)
      for (int q = (kk > kSt ? kk - kSt : 0); q < kk; ++q) mbar_wait(bar(FULL + q % kSt), (q / kSt) & 1);
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc_i8(128, NT);
    const uint64_t a_desc = smem_desc(base, 16, 1024, 2);
    const uint64_t b_desc = smem_desc(kRows ? smem_u32(blocks) : base + 128 * kBK, 16, 1024, 2);
    int kk = 0;
    bool go = true;
    if constexpr (kRows) go = warp_wait(bar(ROWS), 0, s_abort, p.status);
    for (int kb = kb0; go && kb < kb1; ++kb, ++kk) {
      const int s = kk % kSt;
      if (!warp_wait(bar(FULL + s), (kk / kSt) & 1, s_abort, p.status)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = a_desc + uint64_t(s * (kSb >> 4));
        const uint64_t b = b_desc + uint64_t(kRows ? kk * (kRowsM * kBK >> 4) : s * (kSb >> 4));
#pragma unroll
        for (int q = 0; q < kBK / 32; ++q)
          umma_i8(tmem, a + uint64_t(2 * q), b + uint64_t(2 * q), idesc, (kk | q) != 0 ? 1u : 0u);
        umma_commit(bar(EMPTY + s));
      }
      __syncwarp();
    }
    if (elect_one()) umma_commit(bar(ACC));  // also when unwinding: every issued MMA finishes before TMEM is released
    __syncwarp();
  } else {
    if constexpr (kRows) {
      if (p.vec_rows) quantize_share<T, true>(p, blocks, s_top, s_scale, kb0, kb1, warp - 2, lane);
      else quantize_share<T, false>(p, blocks, s_top, s_scale, kb0, kb1, warp - 2, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(ROWS));
    }
    // the CTA's partial sums, (token, channel) int32, into the ring once every MMA has read it
    const int quad = warp & 3, half = (warp - 2) >> 2;
    if (warp_wait(bar(ACC), 0, s_abort, p.status)) {
      tc_fence_after();
      int32_t* acc = reinterpret_cast<int32_t*>(gbase) + quad * 32 + lane;
#pragma unroll
      for (int c = half; c < NT / 16; c += 2) {
        float v[16];
        tmem_ld16(tmem + (uint32_t(quad * 32) << 16) + c * 16, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[(c * 16 + i) * 128] = __float_as_int(v[i]);
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  const bool bad = aborted(s_abort);
  cluster_sync();  // every CTA's partial sums are in place
  if (warp >= 2 && !bad) {
    // tokens [NT rank / S, NT (rank + 1) / S), two per warp at a time, four channels a lane;
    // all parts of both are on their way before the first is added
    const T* bias = static_cast<const T*>(p.bias);
    T* y = static_cast<T*>(p.y);
    const int32_t ch = n0 + lane * 4;
    float ws[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = ch + i < p.n;
      ws[i] = in ? __ldg(p.w_scale + ch + i) : 0.f;
      b[i] = in && bias != nullptr ? DT<T>::to_f(bias[ch + i]) : 0.f;
    }
    const bool whole = ch + 3 < p.n && p.tma_out;
    const int t_end = NT * (rank + 1) / S;
    uint32_t part[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) part[r] = mapa_shared(base + uint32_t(lane) * 16u, uint32_t(r < S ? r : 0));
    for (int t = NT * rank / S + (warp - 2); t < t_end && m0 + t < p.m_rows; t += 2 * kSplitEpiWarps) {
      const int t2 = t + kSplitEpiWarps;
      const bool two = t2 < t_end && m0 + t2 < p.m_rows;
      int4 v[2][8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        v[0][r] = v[1][r] = make_int4(0, 0, 0, 0);
        if (r < S) {
          v[0][r] = ld_dsmem_i4(part[r] + uint32_t(t) * 512u);
          if (two) v[1][r] = ld_dsmem_i4(part[r] + uint32_t(t2) * 512u);
        }
      }
      float xs[2];
      if constexpr (kRows) {
        xs[0] = s_scale[t];
        xs[1] = two ? s_scale[t2] : 0.f;
      } else {
        xs[0] = __ldg(p.x_scale + m0 + t);
        xs[1] = two ? __ldg(p.x_scale + m0 + t2) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (k == 1 && !two) break;
        int4 a = v[k][0];
#pragma unroll
        for (int r = 1; r < 8; ++r) {
          a.x += v[k][r].x;
          a.y += v[k][r].y;
          a.z += v[k][r].z;
          a.w += v[k][r].w;
        }
        const float2 lo = finish2<T, kAct>(a.x, a.y, f2(xs[k]), make_float2(ws[0], ws[1]), make_float2(b[0], b[1]));
        const float2 hi = finish2<T, kAct>(a.z, a.w, f2(xs[k]), make_float2(ws[2], ws[3]), make_float2(b[2], b[3]));
        T* dst = y + (m0 + (k == 0 ? t : t2)) * p.ldy + ch;
        if (whole) {
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(dst) = make_uint2(Pack2<T>::pack(lo.x, lo.y), Pack2<T>::pack(hi.x, hi.y));
          else
            *reinterpret_cast<float4*>(dst) = make_float4(lo.x, lo.y, hi.x, hi.y);
        } else {
          const float o[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (ch + i < p.n) dst[i] = DT<T>::from_f(o[i]);
        }
      }
    }
  }
  tc_fence_before();
  cluster_sync();  // no CTA leaves while a peer may still read its partial sums
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, kTmemCols);
  }
}

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

int encode(CUtensorMap* map, CUtensorMapDataType dt, int es, const void* base, int64_t cols, int64_t rows, int64_t ld,
           int box_cols, int box_rows, CUtensorMapSwizzle swz, const char* what) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (enc == nullptr) return set_error(LF_ERR_DRIVER, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(ld) * cuuint64_t(es)};
  const cuuint32_t box[2] = {cuuint32_t(box_cols), cuuint32_t(box_rows)}, estr[2] = {1, 1};
  const CUresult r = enc(map, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(LF_ERR_CUDA, "lf_linear_int8: cuTensorMapEncodeTiled(%s) failed: %d", what, int(r));
  return LF_OK;
}

template <auto Kern>
int launch_cluster(const char* what, dim3 grid, int threads, int smem, int cluster, int dev, cudaStream_t s,
                   const LinearInt8Params& p) {
  cudaError_t e = allow_smem<Kern>(dev, smem);
  if (e != cudaSuccess) return cuda_error(e, what);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, Kern, p);
  if (e != cudaSuccess) return cuda_error(e, what);
  count_launch();
  return LF_OK;
}

template <typename T, int kAct>
int launch_batch(LinearInt8Params& p, int dev, cudaStream_t s) {
  p.n_tiles_n = (p.n + kBN - 1) / kBN;
  const int64_t tiles = (p.m_rows + 2 * kBM - 1) / (2 * kBM) * p.n_tiles_n;
  if (tiles > INT32_MAX / 2) return set_error(LF_ERR_UNSUPPORTED, "lf_linear_int8: %lld output tiles", (long long)tiles);
  p.n_tiles = int32_t(tiles);
  const int pairs = device_sms(dev) / 2;
  const unsigned grid = unsigned(2 * (p.n_tiles < pairs ? p.n_tiles : pairs));
  return launch_cluster<linear_int8_kernel<T, kAct>>("launch linear_int8", dim3(grid), kThreads, smem_bytes(sizeof(T)),
                                                     2, dev, s, p);
}

template <typename T, int NT, int kAct, bool kRows = false>
int launch_split(LinearInt8Params& p, int dev, cudaStream_t s) {
  p.n_tiles_n = (p.n + 127) / 128;
  const dim3 grid(unsigned(p.n_tiles_n) * unsigned(p.split), unsigned((p.m_rows + NT - 1) / NT));
  return launch_cluster<linear_int8_split_kernel<T, NT, kAct, kRows>>("launch linear_int8_split", grid, kSplitThreads,
                                                                      kRows ? rows_smem_bytes() : split_smem_bytes(NT),
                                                                      p.split, dev, s, p);
}

template <typename T, int kAct>
int launch(LinearInt8Params& p, bool batch, int nt, int dev, cudaStream_t s) {
  if (batch) return launch_batch<T, kAct>(p, dev, s);
  if (p.rows != nullptr) return launch_split<T, kRowsM, kAct, true>(p, dev, s);
  if (nt == 16) return launch_split<T, 16, kAct>(p, dev, s);
  if (nt == 32) return launch_split<T, 32, kAct>(p, dev, s);
  if (nt == 64) return launch_split<T, 64, kAct>(p, dev, s);
  return launch_split<T, 128, kAct>(p, dev, s);
}

}  // namespace

}  // namespace lf

using namespace lf;

namespace {

// x in 8-bit integers with x_scale, or (float_rows) rows of dtype that one launch quantises too.
int run(const char* fn, void* stream, int dtype, const void* x, int64_t ldx, const float* x_scale, bool float_rows,
        const int8_t* w, int64_t ldw, const float* w_scale, const void* bias, void* y, int64_t ldy, int64_t m, int n,
        int k, int act, int32_t* status) {
  if (dtype != LF_DTYPE_BF16 && dtype != LF_DTYPE_F16 && dtype != LF_DTYPE_F32)
    return set_error(LF_ERR_INVALID, "%s: unknown dtype %d", fn, dtype);
  if (act != LF_ACT_NONE && act != LF_ACT_GELU) return set_error(LF_ERR_INVALID, "%s: unknown act %d", fn, act);
  if (m < 0 || m > INT32_MAX - 256 || n <= 0 || n > INT32_MAX - 256 || k <= 0)
    return set_error(LF_ERR_INVALID, "%s: m %lld, n %d, k %d", fn, (long long)m, n, k);
  if (k > 131072) return set_error(LF_ERR_UNSUPPORTED, "%s: k %d above 131072 (the sum could leave 32 bits)", fn, k);
  if (m == 0) return LF_OK;
  if (x == nullptr || (x_scale == nullptr && !float_rows) || w == nullptr || w_scale == nullptr || y == nullptr)
    return set_error(LF_ERR_INVALID, "%s: null x, w, scales or y", fn);
  if (ldx < k || ldw < k || ldy < n) return set_error(LF_ERR_INVALID, "%s: a row stride is below its row", fn);
  if (!aligned16(w) || ldw % 16 != 0 || (!float_rows && (!aligned16(x) || ldx % 16 != 0)))
    return set_error(LF_ERR_INVALID, "%s: 8-bit x and w need 16-byte aligned rows", fn);
  const int es = dtype == LF_DTYPE_F32 ? 4 : 2;
  LinearInt8Params p;
  memset(&p, 0, sizeof(p));
  p.x_scale = x_scale;
  p.w_scale = w_scale;
  p.bias = bias;
  p.y = y;
  p.ldy = ldy;
  p.m_rows = m;
  p.n = n;
  p.n_kb = (k + kBK - 1) / kBK;
  p.tma_out = aligned16(y) && (ldy * es) % 16 == 0 ? 1 : 0;
  p.vec_ch = (reinterpret_cast<uintptr_t>(w_scale) & 7u) == 0 && (reinterpret_cast<uintptr_t>(bias) & (2u * es - 1u)) == 0;
  p.status = status;
  if (float_rows) {
    p.rows = x;
    p.ld_rows = ldx;
    p.k = k;
    p.vec_rows = k % 8 == 0 && aligned16(x) && (ldx * es) % 16 == 0;
  }

  // 256 x 256 tiles once a quarter as many as SMs, unless few tokens leave them mostly empty
  // and 128 channels a CTA still find an SM each; below that 128 channels x nt tokens.
  // Measured with the few-token kernel and with the other (us, bf16, no activation):
  //   n 1,024, k 4,096: 512 tokens (8 tiles) 14.3 and 20.5; 2,048 (32) 18.5 and 20.5;
  //     3,000 (48) 32.8 and 20.5
  //   n 4,096, k 1,024: 256 tokens (16) 12.3 both; 512 (32) 14.3 both; 1,024 (64) 24.6 and 14.3
  //   n 10,240, k 2,560: 256 tokens (40) 26.6 and 16.4
  // and without launch: n 10,240, k 2,560: 16 tokens 8.4 and 12.8, 64 10.0 and 11.1, 128 11.6 and
  // 11.4; n 40,960: 64 tokens 32.9 and 25.6
  const int dev = current_device(), sms = device_sms(dev);
  const int64_t big = ((m + 255) / 256) * ((n + 255) / 256);
  const bool batch = big > sms / 4 && !(m <= 64 && (n + 127) / 128 <= sms) && !float_rows;
  const int nt = batch ? 128 : m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
  p.split = 1;
  if (!batch) {
    const int64_t tiles = ((m + nt - 1) / nt) * ((n + 127) / 128);
    // K is split while every cluster still has its place at once: the GPU's processing clusters
    // leave room for 33 clusters of four such CTAs and 15 of eight on 148 SMs (16 of eight: 20.5 us,
    // as 8 with K whole in a quarter each 14.3; 256 tokens, n 1,024, k 4,096).
    const int64_t room[3] = {sms, int64_t(sms) * 9 / 10, int64_t(sms) * 13 / 16};  // in CTAs, clusters of 2, 4, 8
    for (int i = 0; i < 3 && tiles * p.split * 2 <= room[i] && p.split * 2 <= p.n_kb; ++i) p.split *= 2;
  }
  int rc;
  if (!float_rows &&
      (rc = encode(&p.x_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, k, m, ldx, kBK, nt, CU_TENSOR_MAP_SWIZZLE_128B, "x")))
    return rc;
  if ((rc = encode(&p.w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, k, n, ldw, kBK, 128, CU_TENSOR_MAP_SWIZZLE_128B, "w")))
    return rc;
  if (batch && p.tma_out) {
    const CUtensorMapDataType dt = dtype == LF_DTYPE_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : dtype == LF_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    if ((rc = encode(&p.y_map, dt, es, y, n, m, ldy, kOutCols, 32,
                     es == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, "y")))
      return rc;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    return act == LF_ACT_GELU ? launch<T, LF_ACT_GELU>(p, batch, nt, dev, s) : launch<T, LF_ACT_NONE>(p, batch, nt, dev, s);
  };
  if (dtype == LF_DTYPE_BF16) return go(__nv_bfloat16{});
  if (dtype == LF_DTYPE_F16) return go(__half{});
  return go(float{});
}

}  // namespace

namespace lf {

// One launch or two, GPU time of calls in a row (us, bf16, n 1,024; a launch saves the host
// 4.5 us besides): k 1,024: 1 row 4.4 and 5.0, 8 4.7 and 5.1, 16 5.6 and 5.1; k 4,096: 1 row 4.9
// and 5.1, 4 5.4 and 5.4, 8 6.2 and 5.4, 16 8.2 and 5.5 (every CTA reads all rows).
bool linear_int8_takes_rows(int64_t m, int k) { return m <= kRowsM && k <= kRowsK && m * k <= 16384; }

int linear_int8_rows(void* stream, int dtype, const void* x, int64_t ldx, const int8_t* w, int64_t ldw,
                     const float* w_scale, const void* bias, void* y, int64_t ldy, int64_t m, int n, int k, int act,
                     int32_t* status) {
  return run("lf_linear_rows_int8", stream, dtype, x, ldx, nullptr, true, w, ldw, w_scale, bias, y, ldy, m, n, k, act, status);
}

}  // namespace lf

extern "C" int lf_linear_int8(void* stream, int dtype, const int8_t* x, int64_t ldx, const float* x_scale,
                              const int8_t* w, int64_t ldw, const float* w_scale, const void* bias, void* y,
                              int64_t ldy, int64_t m, int n, int k, int act, int32_t* status) {
  return run("lf_linear_int8", stream, dtype, x, ldx, x_scale, false, w, ldw, w_scale, bias, y, ldy, m, n, k, act, status);
}
