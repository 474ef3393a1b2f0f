// Cross attention of packed sequences: the queries of sequence s attend to the keys and
// values of that sequence's encoder states, which have a length of their own:
//     out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / group]) v[j, h / group]
// over the sequence's keys j (group query heads share a key head).  A sequence without
// keys gives zeros.  head_dim is a multiple of 8 up to 128; the kernels are compiled for
// 64 and 128 columns and read only the head's own (tensor maps and loads end at
// head_dim, the columns past it count as zeros and cost no memory traffic).
//
// Softmax statistics and sums are f32, in the log2 domain; the unnormalised
// probabilities are rounded to the 16-bit type for the second product, as the tensor
// cores take them (each is within half a step of its value, and the sum that divides
// them is taken before the rounding).  Keys past a sequence's end are never multiplied:
// their scores are replaced, and their value rows are zeroed on chip, so that infinities
// or NaN in a neighbouring sequence's states do not reach this one.
//
// Two kernels:
//
// cross_decode_kernel, for few query rows (single tokens), where reading K and V once at
// HBM speed is the bound.  One CTA per (sequence, key head, block of query rows, share of
// the keys): its rows are the group's heads and the sequence's queries, 16 of them (one
// mma.sync tile; two tiles a CTA took 166 registers and measured slower than two CTAs side
// by side, 59 against 46 us), so K and V are read once for all of them.  Four warps take 16-key tiles
// in turn, each with its own ring of asynchronous copies and its own running maximum and
// sum, merged at the end through shared memory.  The keys of a sequence are split over a
// cluster of up to 8 CTAs when there are too few sequences and heads to fill the GPU, or
// to even out long and short ones; the cluster joins its parts through distributed
// shared memory in rank order, so there is no workspace, no second launch and no atomic.
//
// cross_prompt_kernel, for many query rows, on tcgen05.  Work unit = (128 queries of a
// sequence, head).  A persistent CTA per SM runs two groups side by side, each walking
// units of its own with its own warps, rings, barriers and TMEM columns, so that one
// group's exponentials fill the other's waits and neither waits for the other:
//   warps 0-1   producers, one per group: Q, K and V tiles by TMA (SW128 blocks of 64 columns);
//   warps 2-3   MMA issuers, one per group: S = Q K^T, then O += P V of the tile before;
//   warps 4-7,  softmax, one thread per query row.  The row's scores are read from TMEM once
//   8-11        into registers (the first warpgroup hands registers over) and the S buffer
//               is free for the next tile at once; the probabilities go to TMEM columns of
//               their own, from where the second product takes them as its operand.
// With 64 columns a key tile has 128 keys, with 128 columns 64: S, P and O of a group take
// 256 (224) TMEM columns.  A tile's exponentials take the SFU 1,024 (512) clocks, its
// products the tensor cores half as long.  Neither is the bound: over long prompts (8 x 256 to
// 1,024 queries, 1,024 to 8,192 keys, 16 heads of 64: 148 to 159 us) the SFU is busy 53% of
// the time and the tensor pipe 28%; the rest goes to score loads, conversions, sums and waits.
// Every wait is bounded: a timeout sets LF_STATUS_TIMEOUT and the roles unwind.
#include <cmath>
#include <cstring>

#include "lf_common.cuh"
#include "lf_internal.h"

namespace lf {

namespace {

struct alignas(64) CrossParams {
  CUtensorMap q_map, k_map, v_map;  // prompt: 3D {head_dim, heads, rows}, box {64, 1, 128 or the key tile}
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv, n_q, n_kv;
  int32_t n_heads, n_kv_heads, group, d;
  const int4* items;   // two per record: {q_start, q_len, kv_start, kv_len}, {q_tile, 0, 0, 0}
  int32_t n_items;
  int32_t max_q;       // no record's q_len is above it
  int32_t row_blocks;  // decode: CTAs that share a key head's query rows
  int32_t split;       // decode: CTAs of the cluster that share a sequence's keys
  float scale_log2;    // scale * log2(e)
  void* out;
  int64_t ldo;
  int32_t* status;
};

// A record, checked against the tensors and the call: one that names rows outside them, more
// queries than max_q, or a tile past its queries, is reported and stores nothing.
struct Rec {
  int q0, nq, k0, nk, tile;
  bool ok;
};
__device__ __forceinline__ Rec read_rec(const CrossParams& p, int i) {
  const int4 a = __ldg(p.items + 2 * i), b = __ldg(p.items + 2 * i + 1);
  Rec r{a.x, a.y, a.z, a.w, b.x, true};
  r.ok = r.q0 >= 0 && r.nq >= 0 && r.nq <= p.max_q && int64_t(r.q0) + r.nq <= p.n_q && r.k0 >= 0 && r.nk >= 0 &&
         int64_t(r.k0) + r.nk <= p.n_kv && r.tile >= 0 && (r.nq == 0 ? r.tile == 0 : int64_t(r.tile) * 128 < r.nq);
  return r;
}

// ---------------------------------------------------------------------------
// few query rows
// ---------------------------------------------------------------------------
constexpr int kDecodeWarps = 4;
constexpr int kDecodeRows = 16;  // query rows of a CTA: one mma.sync tile
constexpr int kKeyTile = 16;  // keys a warp takes at a time

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes to shared memory, or 16 zeros when `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ float ld_dsmem_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// three stages a warp: with four, three CTAs of 64 columns fit an SM instead of four (64
// sequences of 4,096 keys, 16 heads: 185 us against 159)
__host__ __device__ constexpr int decode_stages(int) { return 3; }
__host__ __device__ constexpr int decode_pitch(int kd) { return kd + 8; }  // f32 columns of a partial output row
// [Q tile][ring, reused for the warps' partial outputs][warps' m and l][the CTA's m and l]
__host__ __device__ constexpr int decode_q_bytes(int kd) { return kDecodeRows * kd * 2; }
__host__ __device__ constexpr int decode_ring_bytes(int kd) {
  return kDecodeWarps * decode_stages(kd) * 2 * kKeyTile * kd * 2;
}
__host__ __device__ constexpr int decode_smem(int kd) {
  return decode_q_bytes(kd) + decode_ring_bytes(kd) + (kDecodeWarps + 1) * kDecodeRows * 2 * 4;
}
static_assert(kDecodeWarps * kDecodeRows * decode_pitch(64) * 4 <= decode_ring_bytes(64), "partial outputs reuse the ring");
static_assert(kDecodeWarps * kDecodeRows * decode_pitch(128) * 4 <= decode_ring_bytes(128), "partial outputs reuse the ring");

template <typename T, int kD>
__global__ void __launch_bounds__(32 * kDecodeWarps) cross_decode_kernel(const __grid_constant__ CrossParams p) {
  constexpr int kSt = decode_stages(kD), kTile = kKeyTile * kD * 2, kCh = kD / 8, kPitch = decode_pitch(kD);
  constexpr int kRowsMax = kDecodeRows;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.split;
  const int rank = S > 1 ? int(cluster_ctarank()) : 0;
  // a unit's row blocks lie side by side: they read the same keys at the same time
  const int unit = int(blockIdx.x) / (S * p.row_blocks), row_block = int(blockIdx.x) / S % p.row_blocks;
  const int kvh = unit % p.n_kv_heads;
  const uint32_t sQ = smem_u32(smem);
  const uint32_t ring = sQ + decode_q_bytes(kD) + warp * (kSt * 2 * kTile);
  float* s_part = reinterpret_cast<float*>(smem + decode_q_bytes(kD));
  float* s_ml = s_part + decode_ring_bytes(kD) / 4;  // [warp][row]{m, l}, then the CTA's

  pdl_wait();
  pdl_launch_dependents();

  const Rec rec = read_rec(p, unit / p.n_kv_heads);
  // the cluster's CTAs share the record, so they leave together
  if (!rec.ok || rec.tile != 0) {
    if (tid == 0) set_status(p.status, LF_STATUS_BAD_SEGMENT);
    return;
  }
  const int row0 = row_block * kRowsMax;
  const int rows = min(kRowsMax, rec.nq * p.group - row0);  // row r: query (row0 + r) / group, head (row0 + r) % group
  if (rows <= 0) return;
  const int nch = p.d / 8;              // 16-byte chunks of a head's row
  const int nks = (p.d + 15) / 16;      // 16-column steps

  // chunk c of a row sits at c ^ (row & 7) within its 128-byte line, so that ldmatrix's
  // eight rows fall into different banks
  auto at = [](uint32_t base, int row, int c) { return base + uint32_t(row * (kD * 2) + ((c ^ (row & 7)) << 4)); };

  const T* qg = static_cast<const T*>(p.q);
  for (int i = tid; i < kRowsMax * kCh; i += 32 * kDecodeWarps) {
    const int r = i / kCh, c = i % kCh;
    const bool in = r < rows && c < nch;
    const int rr = row0 + (in ? r : 0);
    const T* src = qg + int64_t(rec.q0 + rr / p.group) * p.ldq + int64_t(kvh * p.group + rr % p.group) * p.d + (in ? c : 0) * 8;
    cp_async16(at(sQ, r, c), src, in ? 16u : 0u);
  }
  cp_async_commit();

  // this CTA's 16-key tiles, every fourth one this warp's
  const int n_tiles = (rec.nk + kKeyTile - 1) / kKeyTile;
  const int t0 = int(int64_t(n_tiles) * rank / S), t1 = int(int64_t(n_tiles) * (rank + 1) / S);
  const int n_my = t1 - t0 > warp ? (t1 - t0 - warp + kDecodeWarps - 1) / kDecodeWarps : 0;
  // Addresses are kept as what changes from one copy to the next: a lane copies chunk
  // lane % kCh of rows kRowsJ apart, whose swizzled places repeat every kPeriod copies.
  constexpr int kRowsJ = 32 / kCh, kPeriod = 8 / kRowsJ, kCopies = kKeyTile / kRowsJ;
  const int my_row = lane / kCh, my_ch = lane % kCh;
  const bool my_col = my_ch < nch;  // a chunk past the head is never copied: zeros, written once
  uint32_t cp_off[kPeriod];
#pragma unroll
  for (int x = 0; x < kPeriod; ++x) cp_off[x] = at(0, x * kRowsJ + my_row, my_ch);
  const T* kp = static_cast<const T*>(p.k) + (int64_t(rec.k0) + (t0 + warp) * kKeyTile + my_row) * p.ldk + int64_t(kvh) * p.d + my_ch * 8;
  const T* vp = static_cast<const T*>(p.v) + (int64_t(rec.k0) + (t0 + warp) * kKeyTile + my_row) * p.ldv + int64_t(kvh) * p.d + my_ch * 8;
  if (nch < kCh) {
    for (int i = lane; i < kSt * 2 * kKeyTile * (kCh - nch); i += 32) {
      const int r = i / (kCh - nch), c = nch + i % (kCh - nch);  // the stages' tiles lie one after the other
      *reinterpret_cast<uint4*>(smem + (at(ring, r, c) - sQ)) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  int issued = 0;
  uint32_t st_issue = ring;
  auto issue = [&]() {  // the next tile's copies into the next stage
    if (issued < n_my) {
      const int left = rec.nk - (t0 + warp + kDecodeWarps * issued) * kKeyTile;
      if (my_col) {
        if (left >= kKeyTile) {
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            const uint32_t dst = st_issue + cp_off[j % kPeriod] + (j / kPeriod) * (8 * kD * 2);
            cp_async16(dst, kp + j * kRowsJ * p.ldk, 16u);
            cp_async16(dst + kTile, vp + j * kRowsJ * p.ldv, 16u);
          }
        } else {  // rows past the end become zeros
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            const uint32_t dst = st_issue + cp_off[j % kPeriod] + (j / kPeriod) * (8 * kD * 2);
            const bool in = j * kRowsJ + my_row < left;
            cp_async16(dst, in ? kp + j * kRowsJ * p.ldk : static_cast<const T*>(p.k), in ? 16u : 0u);
            cp_async16(dst + kTile, in ? vp + j * kRowsJ * p.ldv : static_cast<const T*>(p.v), in ? 16u : 0u);
          }
        }
        kp += kDecodeWarps * kKeyTile * p.ldk;
        vp += kDecodeWarps * kKeyTile * p.ldv;
      }
      ++issued;
      st_issue = st_issue == ring + (kSt - 1) * (2 * kTile) ? ring : st_issue + 2 * kTile;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kSt - 1; ++i) issue();
  cp_async_wait<kSt - 1>();  // Q has landed
  __syncthreads();

  uint32_t qf[kD / 16][4];
#pragma unroll
  for (int ks = 0; ks < kD / 16; ++ks) ldsm4(qf[ks], at(sQ, (lane & 7) + ((lane >> 3) & 1) * 8, ks * 2 + (lane >> 4)));
  float o[kD / 8][4] = {};
  float mrow[2] = {-INFINITY, -INFINITY}, lrow[2] = {0.f, 0.f};

  // ldmatrix rows: K {keys 0-7, 8-15} x {8 columns, next 8}, V the other way round; chunk
  // 2 ks + x of 16-column step ks repeats its swizzle every four steps (128 bytes)
  uint32_t k_off[4], v_off[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    k_off[ks] = at(0, (lane & 7) + (lane >> 4) * 8, ks * 2 + ((lane >> 3) & 1));
    v_off[ks] = at(0, (lane & 7) + ((lane >> 3) & 1) * 8, ks * 2 + (lane >> 4)) + kTile;
  }
  uint32_t st = ring;
  for (int i = 0; i < n_my; ++i) {
    cp_async_wait<kSt - 2>();
    __syncwarp();
    float s[2][4] = {}, s1[2][4] = {};  // even and odd steps: half as long a chain of products
#pragma unroll
    for (int ks = 0; ks < kD / 16; ++ks) {
      if (ks >= nks) break;
      uint32_t kf[4];
      ldsm4(kf, st + k_off[ks & 3] + (ks >> 2) * 128);
      mma16816<T>(ks & 1 ? s1[0] : s[0], qf[ks], kf[0], kf[1]);
      mma16816<T>(ks & 1 ? s1[1] : s[1], qf[ks], kf[2], kf[3]);
    }
    const int left = rec.nk - (t0 + warp + kDecodeWarps * i) * kKeyTile;  // keys of the sequence from this tile on
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[n][x] += s1[n][x];
        if (n * 8 + (lane & 3) * 2 + (x & 1) >= left) s[n][x] = -INFINITY;
      }
    uint32_t pf[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // rows lane / 4 and lane / 4 + 8
      if (h * 8 >= rows) {  // eight rows without a query
        pf[h] = pf[2 + h] = 0u;
        continue;
      }
      float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(mrow[h], mx * p.scale_log2);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;  // every score so far is -inf: p = 0
      if (__any_sync(0xffffffffu, m_new != mrow[h])) {
        const float alpha = sfu_ex2(mrow[h] - m_use);
        mrow[h] = m_new;
        lrow[h] *= alpha;
#pragma unroll
        for (int n = 0; n < kD / 8; ++n) {
          o[n][2 * h] *= alpha;
          o[n][2 * h + 1] *= alpha;
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float e0 = sfu_ex2(fmaf(s[n][2 * h], p.scale_log2, -m_use));
        const float e1 = sfu_ex2(fmaf(s[n][2 * h + 1], p.scale_log2, -m_use));
        lrow[h] += e0 + e1;
        pf[2 * n + h] = Pack2<T>::pack(e0, e1);
      }
    }
#pragma unroll
    for (int ks = 0; ks < kD / 16; ++ks) {
      if (ks >= nks) break;
      uint32_t vf[4];
      ldsm4_t(vf, st + v_off[ks & 3] + (ks >> 2) * 128);
      mma16816<T>(o[2 * ks], pf, vf[0], vf[1]);
      mma16816<T>(o[2 * ks + 1], pf, vf[2], vf[3]);
    }
    issue();  // into the stage of tile i - 1, which every lane has left
    st = st == ring + (kSt - 1) * (2 * kTile) ? ring : st + 2 * kTile;
  }
  cp_async_wait<0>();
  __syncthreads();  // every warp is done with the ring

  // the warps' parts: output rows, maximum and sum
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = h * 8 + (lane >> 2);
    float l = lrow[h];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* dst = s_part + (warp * kRowsMax + r) * kPitch + (lane & 3) * 2;
#pragma unroll
    for (int n = 0; n < kD / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    if ((lane & 3) == 0) {
      s_ml[(warp * kRowsMax + r) * 2] = mrow[h];
      s_ml[(warp * kRowsMax + r) * 2 + 1] = l;
    }
  }
  __syncthreads();
  T* out = static_cast<T*>(p.out);
  auto store = [&](int r, int c4, float4 v, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int rr = row0 + r;
    T* dst = out + int64_t(rec.q0 + rr / p.group) * p.ldo + int64_t(kvh * p.group + rr % p.group) * p.d + c4 * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(Pack2<T>::pack(v.x * inv, v.y * inv), Pack2<T>::pack(v.z * inv, v.w * inv));
  };
  // n parts of one row: their joint maximum, and part i's weight 2^(m_i - max) (0 without keys)
  float* s_cta = s_ml + kDecodeWarps * kRowsMax * 2;
  const int c4s = p.d / 4;
  for (int i = tid; i < rows * c4s; i += 32 * kDecodeWarps) {
    const int r = i / c4s, c4 = i % c4s;
    float mw[kDecodeWarps], mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      mw[w] = s_ml[(w * kRowsMax + r) * 2];
      mx = fmaxf(mx, mw[w]);
    }
    const float m_use = mx == -INFINITY ? 0.f : mx;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      const float f = sfu_ex2(mw[w] - m_use);
      const float4 v = *reinterpret_cast<const float4*>(s_part + (w * kRowsMax + r) * kPitch + c4 * 4);
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
      l += s_ml[(w * kRowsMax + r) * 2 + 1] * f;
    }
    if (S == 1) {
      store(r, c4, acc, l);
    } else {  // the CTA's part replaces warp 0's (only this thread reads it)
      *reinterpret_cast<float4*>(s_part + r * kPitch + c4 * 4) = acc;
      if (c4 == 0) {
        s_cta[2 * r] = mx;
        s_cta[2 * r + 1] = l;
      }
    }
  }
  if (S == 1) return;
  cluster_sync();
  const uint32_t a_part = smem_u32(s_part), a_cta = smem_u32(s_cta);
  for (int i = rank * 32 * kDecodeWarps + tid; i < rows * c4s; i += S * 32 * kDecodeWarps) {
    const int r = i / c4s, c4 = i % c4s;
    float mx = -INFINITY;
    for (int t = 0; t < S; ++t) mx = fmaxf(mx, ld_dsmem_f32(mapa_shared(a_cta + 8 * r, t)));
    const float m_use = mx == -INFINITY ? 0.f : mx;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int t = 0; t < S; ++t) {
      const float f = sfu_ex2(ld_dsmem_f32(mapa_shared(a_cta + 8 * r, t)) - m_use);
      const float4 v = ld_dsmem_f4(mapa_shared(a_part + uint32_t(r * kPitch + c4 * 4) * 4u, t));
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
      l += ld_dsmem_f32(mapa_shared(a_cta + 8 * r + 4, t)) * f;
    }
    store(r, c4, acc, l);
  }
  cluster_sync();  // no CTA leaves while a peer may still read its part
}

// ---------------------------------------------------------------------------
// many query rows
// ---------------------------------------------------------------------------
constexpr int kRows = 128;     // query tile rows
constexpr int kGroups = 2;
constexpr int kThreads = 128 * (1 + kGroups);
// Registers: the producer / MMA warpgroup gives up what the softmax warpgroups take, so
// that a row's 128 scores stay in registers (128 x 88 + 256 x 208 = 384 x 168, the launch's).
constexpr int kRegsIssue = 88, kRegsSoftmax = 208;
constexpr float kMaxSlack = 8.f;    // log2 units the running max may lag a tile's max
constexpr float kSumSlack = 256.f;  // 2^kMaxSlack

template <int kD>
struct Shape {
  static constexpr int kKeys = kD == 64 ? 128 : 64;   // key tile rows
  static constexpr int kBlocks = kD / 64;             // 64-column SW128 blocks of a head's row
  static constexpr int kQBytes = kRows * kD * 2;
  static constexpr int kKvBytes = kKeys * kD * 2;     // 16 KB
  static constexpr int kStages = kD == 64 ? 3 : 2;    // K stages and V stages of a group
  // TMEM columns of a group: S, then P (two probabilities a column), then O
  static constexpr int kPCol = kKeys, kOCol = kKeys + kKeys / 2;
  static constexpr int kGroupBytes = kQBytes + 2 * kStages * kKvBytes;
  static constexpr int kSmem = 1024 + kGroups * kGroupBytes + 1024;
  static_assert(kOCol + kD <= 256, "TMEM columns of a group");
  static_assert(kSmem <= 232448, "above the 227 KB of shared memory a CTA may use");
};

__device__ __forceinline__ bool aborted(const int32_t* f) { return *reinterpret_cast<const volatile int32_t*>(f) != 0; }

// max(a, b, c) in one instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// D[tmem] (+)= A[tmem] * B[smem desc]: A's row is the TMEM lane, two 16-bit elements a column.
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 128 consecutive TMEM columns of this warp's 32 lanes, both halves in flight at once.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
      "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
      "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
      "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127"
      "}, [%129];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
        "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
        "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
        "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
        "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
        "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
        "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
        "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr), "r"(taddr + 64)
      : "memory");
}

template <int N>
__device__ __forceinline__ void set_max_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_max_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// A unit's record as every role reads it: keys to walk (at least one, so that all roles
// take the same steps), and what is stored: 0 the result, 1 nothing, 2 zeros (no keys).
struct Unit {
  int q0, nq, k0, nk, tile, what;
};

// A group's walk over its units and their key tiles.
struct Cursor {
  int64_t unit;  // global unit index, or >= n_units when done
  Unit it;
  int j, n_kv;   // key tile within the unit
  int u;         // units this group has started (for buffer parities)
  int t;         // tiles this group has started
};

template <typename T, int kD>
__global__ void __launch_bounds__(kThreads, 1) cross_prompt_kernel(const __grid_constant__ CrossParams p) {
  using Sh = Shape<kD>;
  constexpr int kKeys = Sh::kKeys, kKvBytes = Sh::kKvBytes, kStages = Sh::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  // What is the same in a whole warp comes from lane 0 by shuffle, so that the compiler
  // knows it: descriptors, coordinates and barrier addresses then live in uniform
  // registers (long prompts 176 -> 156 us).
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const int grp = warp < 4 ? warp & 1 : (warp - 4) >> 2;  // the group this warp works for

  const uint32_t sQ = base + grp * Sh::kGroupBytes;
  const uint32_t sK = sQ + Sh::kQBytes;
  const uint32_t sV = sK + kStages * kKvBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(gbase + kGroups * Sh::kGroupBytes);
  constexpr int Q_FULL = 0, Q_EMPTY = 1, S_FULL = 2, S_EMPTY = 3, P_FULL = 4, PV_DONE = 5, O_EMPTY = 6, DRAIN = 7,
                K_FULL = 8, K_EMPTY = K_FULL + kStages, V_FULL = K_EMPTY + kStages, V_EMPTY = V_FULL + kStages,
                N_BARS = V_EMPTY + kStages;  // of a group
  auto bar = [&](int i) { return smem_u32(&bars[grp * N_BARS + i]); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(&bars[kGroups * N_BARS]);
  int32_t* s_abort = reinterpret_cast<int32_t*>(tmem_slot + 1);
  const int64_t n_units = int64_t(p.n_items) * p.n_heads;

  if (warp < kGroups && lane == 0) {  // each producer warp: its group's barriers
    for (int i = 0; i < N_BARS; ++i) mbar_init(bar(i), i == S_EMPTY || i == P_FULL || i == O_EMPTY ? 4 : 1);
    if (warp == 0) *s_abort = 0;
    fence_mbar_init();
    prefetch_tmap(&p.q_map);
    prefetch_tmap(&p.k_map);
    prefetch_tmap(&p.v_map);
  }
  if (warp == 2) {
    __syncwarp();
    tmem_alloc(smem_u32(tmem_slot), 512);
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot) + uint32_t(grp) * 256;
  pdl_wait();
  pdl_launch_dependents();

  // by a whole warp, and by one lane
  auto wwait = [&](uint32_t b, uint32_t parity) { return warp_wait(b, parity, s_abort, p.status); };
  auto wait = [&](uint32_t b, uint32_t parity) {
    if (mbar_try_wait(b, parity)) return true;
    if (aborted(s_abort)) return false;
    if (mbar_wait(b, parity)) return true;
    set_status(p.status, LF_STATUS_TIMEOUT);
    atomicExch(s_abort, 1);
    return false;
  };
  auto unit_of = [&](int64_t unit) {
    const Rec r = read_rec(p, int(unit / p.n_heads));
    if (!r.ok) {
      set_status(p.status, LF_STATUS_BAD_SEGMENT);
      return Unit{0, 0, 0, 1, 0, 1};
    }
    if (r.nq == 0) return Unit{0, 0, 0, 1, 0, 1};
    if (r.nk == 0) return Unit{r.q0, r.nq, 0, 1, r.tile, 2};
    return Unit{r.q0, r.nq, r.k0, r.nk, r.tile, 0};
  };
  // Round i gives every group of every CTA one unit, in the records' order (most keys
  // first), the order of the groups turned round from round to round: a group that had a
  // longer unit gets a shorter one next.
  const int64_t n_slots = int64_t(kGroups) * gridDim.x;
  auto load = [&](Cursor& c) {
    c.j = 0;
    if (c.unit < n_units) {
      const Unit it = unit_of(c.unit);
      c.it = Unit{uniform(it.q0), uniform(it.nq), uniform(it.k0), uniform(it.nk), uniform(it.tile), uniform(it.what)};
      c.n_kv = (c.it.nk + kKeys - 1) / kKeys;
    }
  };
  auto start = [&](Cursor& c) {
    c.unit = blockIdx.x + int64_t(grp) * gridDim.x;
    c.u = c.t = 0;
    load(c);
  };
  auto advance = [&](Cursor& c) {
    ++c.t;
    if (++c.j < c.n_kv) return;
    const int64_t in_round = c.unit - c.u * n_slots;
    ++c.u;
    c.unit = c.u * n_slots + (n_slots - 1 - in_round);
    load(c);
  };
  // A tile of at most 64 queries sits in the upper 64 rows for group 1, so that the two
  // groups' busy warps lie on different schedulers.
  auto shift_of = [&](const Unit& it) { return grp == 1 && it.nq - it.tile * kRows <= 64 ? 64 : 0; };

  if (warp < 4) {
    set_max_regs_dec<kRegsIssue>();
    if (warp < 2) {
      // ------------------------------------------------------------ producer
      Cursor c;
      start(c);
      bool stop = false;
      while (!stop && c.unit < n_units) {
        const int h = int(c.unit % p.n_heads), hk = h / p.group;
        const int s = c.t % kStages;
        const uint32_t ph = ((c.t / kStages) & 1) ^ 1;
        if (c.j == 0) {  // the unit's Q tile, once the previous unit has no S left to issue
          if (!wwait(bar(Q_EMPTY), (c.u & 1) ^ 1)) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(bar(Q_FULL), Sh::kQBytes);
            for (int b = 0; b < Sh::kBlocks; ++b)
              tma_load_3d(sQ + b * (kRows * 128), &p.q_map, bar(Q_FULL), b * 64, h,
                          c.it.q0 + c.it.tile * kRows - shift_of(c.it));
          }
          __syncwarp();
        }
        const int32_t krow = c.it.k0 + c.j * kKeys;
        stop = !wwait(bar(K_EMPTY + s), ph);
        if (stop) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar(K_FULL + s), kKvBytes);
          for (int b = 0; b < Sh::kBlocks; ++b)
            tma_load_3d(sK + s * kKvBytes + b * (kKeys * 128), &p.k_map, bar(K_FULL + s), b * 64, hk, krow);
        }
        __syncwarp();
        stop = !wwait(bar(V_EMPTY + s), ph);
        if (stop) {
          mbar_wait(bar(K_FULL + s), ph ^ 1);  // this tile's K lands; its V was not issued
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(bar(V_FULL + s), kKvBytes);
          for (int b = 0; b < Sh::kBlocks; ++b)
            tma_load_3d(sV + s * kKvBytes + b * (kKeys * 128), &p.v_map, bar(V_FULL + s), b * 64, hk, krow);
        }
        __syncwarp();
        advance(c);
      }
      __syncwarp();
      if (aborted(s_abort)) {  // loads nobody consumed must land before the CTA exits (bounded)
        for (int q = (c.t > kStages ? c.t - kStages : 0); q < c.t; ++q) {
          mbar_wait(bar(K_FULL + q % kStages), (q / kStages) & 1);
          mbar_wait(bar(V_FULL + q % kStages), (q / kStages) & 1);
        }
        const int nq = c.u + (c.unit < n_units && c.j > 0 ? 1 : 0);  // only the latest Q can be unconsumed
        if (nq > 0) mbar_wait(bar(Q_FULL), (nq - 1) & 1);
      }
    } else {
      // ------------------------------------------------------------ MMA issuer
      const int nks = (p.d + 15) / 16;  // 16-column steps of a head's row
      const uint32_t idesc_o = umma_idesc_f16(DT<T>::umma_fmt, kRows, uint32_t(nks) * 16, /*a_mn=*/0, /*b_mn=*/1);
      const uint64_t q_desc = smem_desc(sQ, 16, 1024, 2), k_desc0 = smem_desc(sK, 16, 1024, 2),
                     v_desc0 = smem_desc(sV, kKeys * 128, 1024, 2);
      Cursor c;
      start(c);
      bool prev = false, prev_first = false;  // the tile whose O += P V is still to be issued
      int prev_n16 = 0, prev_t = 0, prev_u = 0;
      while (true) {
        const bool now = c.unit < n_units;
        if (!now && !prev) break;
        bool first = false, last = false;
        int n16 = 0;
        const int t = c.t, u = c.u;
        if (now) {
          const int s = t % kStages;
          if ((c.j == 0 && !wwait(bar(Q_FULL), u & 1)) || !wwait(bar(K_FULL + s), (t / kStages) & 1) ||
              !wwait(bar(S_EMPTY), (t & 1) ^ 1))
            break;
          tc_fence_after();
          // S over the tile's keys, to the next multiple of 16
          first = c.j == 0;
          last = c.j == c.n_kv - 1;
          n16 = (min(kKeys, c.it.nk - c.j * kKeys) + 15) / 16;
          const uint32_t idesc = umma_idesc_f16(DT<T>::umma_fmt, kRows, uint32_t(n16) * 16, 0, 0);
          const uint64_t kd = k_desc0 + uint64_t(s * (kKvBytes >> 4));
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kD / 16; ++i) {  // 16 columns are 32 bytes, 64 of them a block
              if (i < nks)
                umma_f16(tmem, q_desc + uint64_t((i >> 2) * (kRows * 8) + (i & 3) * 2),
                         kd + uint64_t((i >> 2) * (kKeys * 8) + (i & 3) * 2), idesc, i > 0 ? 1u : 0u);
            }
            umma_commit(bar(S_FULL));
            umma_commit(bar(K_EMPTY + s));
            if (last) umma_commit(bar(Q_EMPTY));
          }
          __syncwarp();
          advance(c);
        }
        if (prev) {  // O += P V of the tile before
          const int s = prev_t % kStages;
          if (!wwait(bar(V_FULL + s), (prev_t / kStages) & 1) || (prev_first && !wwait(bar(O_EMPTY), (prev_u & 1) ^ 1)) ||
              !wwait(bar(P_FULL), prev_t & 1))
            break;
          tc_fence_after();
          const uint64_t vd = v_desc0 + uint64_t(s * (kKvBytes >> 4));
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kKeys / 16; ++i) {  // 16 value rows are 2,048 bytes
              if (i < prev_n16)
                umma_f16_ta(tmem + Sh::kOCol, tmem + Sh::kPCol + i * 8, vd + uint64_t(i * 128), idesc_o,
                            (prev_first && i == 0) ? 0u : 1u);
            }
            umma_commit(bar(V_EMPTY + s));
            umma_commit(bar(PV_DONE));
          }
          __syncwarp();
        }
        prev = now;
        prev_first = first;
        prev_n16 = n16;
        prev_t = t;
        prev_u = u;
      }
      __syncwarp();
      if (aborted(s_abort)) {  // every issued MMA must finish before TMEM is released (bounded)
        if (elect_one()) umma_commit(bar(DRAIN));
        __syncwarp();
        mbar_wait(bar(DRAIN), 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax (warps 4..11)
    set_max_regs_inc<kRegsSoftmax>();
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t s_addr = tmem + (uint32_t(quad * 32) << 16);  // this row of S
    const uint32_t p_addr = s_addr + Sh::kPCol, o_addr = s_addr + Sh::kOCol;
    const float2 sl2 = f2(p.scale_log2);
    Cursor c;
    start(c);
    float m = -INFINITY, l = 0.f;
    // A unit's output O / l is stored during the next unit's first tile, whose wait for
    // PV_DONE is the wait for the unit's last O += P V: 1 nothing, 2 zeros (no keys), 0 O / l.
    bool pend = false, pend_rows = false;
    int pend_mode = 1;
    float pend_inv = 0.f;
    T* pend_dst = nullptr;
    auto store_pending = [&](bool done) {
      if (done && pend_rows) {
        tc_fence_after();
#pragma unroll 1
        for (int b = 0; b < 2 * Sh::kBlocks; ++b) {
          uint32_t ov[32];
          tmem_ld32(o_addr + b * 32, ov);
          if (pend_mode != 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (b * 32 + q * 8 >= p.d) break;
              uint4 w;
              if (pend_mode == 2) {  // no keys: zeros, whatever the key row read in their place holds
                w = make_uint4(0u, 0u, 0u, 0u);
              } else {
                w.x = Pack2<T>::pack(__uint_as_float(ov[8 * q + 0]) * pend_inv, __uint_as_float(ov[8 * q + 1]) * pend_inv);
                w.y = Pack2<T>::pack(__uint_as_float(ov[8 * q + 2]) * pend_inv, __uint_as_float(ov[8 * q + 3]) * pend_inv);
                w.z = Pack2<T>::pack(__uint_as_float(ov[8 * q + 4]) * pend_inv, __uint_as_float(ov[8 * q + 5]) * pend_inv);
                w.w = Pack2<T>::pack(__uint_as_float(ov[8 * q + 6]) * pend_inv, __uint_as_float(ov[8 * q + 7]) * pend_inv);
              }
              reinterpret_cast<uint4*>(pend_dst + b * 32)[q] = w;
            }
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(O_EMPTY));
      pend = false;
    };
    while (c.unit < n_units) {
      const int t = c.t, j = c.j;
      const bool last = j == c.n_kv - 1;
      const int nvalid = min(kKeys, c.it.nk - j * kKeys);
      // a warp whose 32 rows hold no query does no softmax (its P rows only feed O rows that
      // are never stored)
      const int shift = shift_of(c.it), n_rows = c.it.nq - c.it.tile * kRows;
      const bool rows_live = quad * 32 + 31 >= shift && quad * 32 < shift + n_rows;
      const bool work = wwait(bar(S_FULL), t & 1);
      tc_fence_after();
      float sum = 0.f, m_new = m, alpha = 1.f;
      // the row's scores, all in registers; a short tile reads its first 64 alone
      uint32_t s[kKeys];
      const bool wide = kKeys == 128 && nvalid > 64;
      if (work && rows_live) {
        if constexpr (kKeys == 128) {
          if (wide) {
            tmem_ld128(s_addr, s);
          } else {
            uint32_t lo[64];
            tmem_ld64(s_addr, lo);
#pragma unroll
            for (int q = 0; q < 64; ++q) s[q] = lo[q], s[64 + q] = 0u;
          }
        } else {
          tmem_ld64(s_addr, s);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(S_EMPTY));  // S has been read: the next may be computed
      bool go = work;  // the previous tile's O += P V has finished: P and O are this warp's
      if (work && rows_live) {
        if (nvalid < kKeys) {  // warp-uniform: keys past the end score -inf, so they do not count
#pragma unroll
          for (int q = 0; q < kKeys; ++q)
            if (q >= nvalid) s[q] = __float_as_uint(-INFINITY);
        }
        // The running maximum only moves when a tile's exceeds it by kMaxSlack, so after the
        // unit's first tile the exponentials start from it at once; no exponential is above
        // 2^kMaxSlack unless their sum is, and a warp that finds a row's so takes the maximum and
        // starts again (long prompts 158 -> 149 us).
        bool exact = j == 0 || __any_sync(0xffffffffu, m == -INFINITY);
        float2 sums[2];
#pragma unroll 1
        while (true) {
          if (exact) {
            float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int q = 0; q < 64; q += 2)
              mxs[(q >> 1) & 3] = max3(mxs[(q >> 1) & 3], __uint_as_float(s[q]), __uint_as_float(s[q + 1]));
            if (wide) {
#pragma unroll
              for (int q = 64; q < kKeys; q += 2)
                mxs[(q >> 1) & 3] = max3(mxs[(q >> 1) & 3], __uint_as_float(s[q]), __uint_as_float(s[q + 1]));
            }
            // the scale is positive: max commutes with it
            const float mx = max3(fmaxf(mxs[0], mxs[1]), mxs[2], mxs[3]) * sl2.x;
            m_new = (j == 0 || mx > m + kMaxSlack) ? mx : m;
            alpha = (j == 0) ? 1.f : sfu_ex2(m - (m_new == -INFINITY ? 0.f : m_new));
            if (j >= 1 && __any_sync(0xffffffffu, alpha != 1.f)) {  // O moves to the new maximum
              go = wwait(bar(PV_DONE), (t & 1) ^ 1);
              if (go) {
                tc_fence_after();
#pragma unroll 1
                for (int b = 0; b < 2 * Sh::kBlocks; ++b) {
                  uint32_t ov[32];
                  tmem_ld32(o_addr + b * 32, ov);
#pragma unroll
                  for (int q = 0; q < 32; ++q) ov[q] = __float_as_uint(__uint_as_float(ov[q]) * alpha);
                  tmem_st32(o_addr + b * 32, ov);
                }
              }
            }
          }
          // p = 2^(s - max), rounded to T, two keys a column; every score so far -inf: p = 0
          const float2 neg_m = f2(m_new == -INFINITY ? 0.f : -m_new);
          sums[0] = sums[1] = make_float2(0.f, 0.f);
#pragma unroll
          for (int hh = 0; hh < kKeys / 64; ++hh) {
            if (hh == 0 || wide) {
              uint32_t w[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const int col = hh * 64 + 2 * i;
                const float2 x = f2_fma(make_float2(__uint_as_float(s[col]), __uint_as_float(s[col + 1])), sl2, neg_m);
                const float2 pr = make_float2(sfu_ex2(x.x), sfu_ex2(x.y));
                sums[i & 1] = f2_add(sums[i & 1], pr);
                w[i] = Pack2<T>::pack(pr.x, pr.y);
              }
              if (hh == 0) go = wwait(bar(PV_DONE), (t & 1) ^ 1);
              if (go) tmem_st32(p_addr + hh * 32, w);
            }
          }
          sum = (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
          if (exact || !__any_sync(0xffffffffu, sum > kSumSlack)) break;
          exact = true;
        }
      } else {
        go = work && wwait(bar(PV_DONE), (t & 1) ^ 1);
      }
      if (pend) store_pending(go);  // PV_DONE was that of the unit before's last tile
      l = (j == 0) ? sum : l * alpha + sum;
      m = m_new;
      // the last 16-key step of a tile that ends inside it multiplies value rows past the
      // sequence's end by p = 0: those rows become zeros first (they may hold NaN)
      if ((nvalid & 15) != 0) {
        const int sv = t % kStages;
        if (go && wwait(bar(V_FULL + sv), (t / kStages) & 1)) {
          const int n_zero = 16 - (nvalid & 15);
          uint8_t* vrow = gbase + (sV + sv * kKvBytes - base) + nvalid * 128;
          for (int i = row; i < n_zero * 8 * Sh::kBlocks; i += kRows) {
            const int b = i / (n_zero * 8), x = i % (n_zero * 8);
            *reinterpret_cast<uint4*>(vrow + b * (kKeys * 128) + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
      }
      // This warp has seen PV_DONE of the tile before, so every warp of the group has arrived
      // for that tile and the MMA warp has seen it: this arrival counts for this tile only.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(P_FULL));
      if (last) {  // the unit's output waits for its last O += P V
        const int r = row - shift;  // row of the query tile
        pend = true;
        pend_rows = rows_live;
        pend_mode = r >= 0 && r < n_rows ? c.it.what : 1;
        pend_inv = l == 0.f ? 0.f : 1.f / l;
        pend_dst = static_cast<T*>(p.out) + (int64_t(c.it.q0) + c.it.tile * kRows + r) * p.ldo + int64_t(c.unit % p.n_heads) * p.d;
      }
      advance(c);
    }
    if (pend) store_pending(wwait(bar(PV_DONE), (c.t - 1) & 1));
  }

  __syncthreads();
  tc_fence_after();
  if (warp == 2) {
    __syncwarp();
    tmem_dealloc(*tmem_slot, 512);
  }
}

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

int encode_rows(CUtensorMap* map, int dtype, const void* base, int64_t ld, int64_t rows, int heads, int d, int box_rows,
                const char* what) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (enc == nullptr) return set_error(LF_ERR_DRIVER, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[3] = {cuuint64_t(d), cuuint64_t(heads), cuuint64_t(rows)};
  const cuuint64_t strides[2] = {cuuint64_t(d) * 2, cuuint64_t(ld) * 2};
  const cuuint32_t box[3] = {64, 1, cuuint32_t(box_rows)}, estr[3] = {1, 1, 1};
  const CUresult r = enc(map, dtype == LF_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(LF_ERR_CUDA, "lf_cross_attention_varlen: cuTensorMapEncodeTiled(%s) failed: %d", what, int(r));
  return LF_OK;
}

template <typename T, int kD>
int launch_decode(const CrossParams& p, int dev, cudaStream_t s) {
  constexpr auto kern = cross_decode_kernel<T, kD>;
  constexpr int smem = decode_smem(kD);
  cudaError_t e = allow_smem<kern>(dev, smem);
  if (e != cudaSuccess) return cuda_error(e, "cudaFuncSetAttribute(cross_decode)");
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(p.split);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.n_items) * unsigned(p.n_kv_heads) * unsigned(p.row_blocks) * unsigned(p.split));
  cfg.blockDim = dim3(32 * kDecodeWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return cuda_error(e, "launch cross_decode");
  count_launch();
  return LF_OK;
}

template <typename T, int kD>
int launch_prompt(const CrossParams& p, int dev, cudaStream_t s) {
  constexpr auto kern = cross_prompt_kernel<T, kD>;
  constexpr int smem = Shape<kD>::kSmem;
  cudaError_t e = allow_smem<kern>(dev, smem);
  if (e != cudaSuccess) return cuda_error(e, "cudaFuncSetAttribute(cross_prompt)");
  const int64_t units = int64_t(p.n_items) * p.n_heads, sms = device_sms(dev);
  e = launch_pdl(kern, dim3(unsigned(units < sms ? units : sms)), dim3(kThreads), smem, s, p);
  if (e != cudaSuccess) return cuda_error(e, "launch cross_prompt");
  count_launch();
  return LF_OK;
}

}  // namespace

}  // namespace lf

using namespace lf;

extern "C" int lf_cross_attention_varlen_total(void* stream, int dtype, const void* q, int64_t ldq, int64_t n_q,
                                               const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t n_kv,
                                               int n_heads, int n_kv_heads, int head_dim, const int32_t* items,
                                               int n_items, int max_q, int max_kv, int64_t total_kv, float scale,
                                               void* out, int64_t ld_out, int32_t* status) {
  const char* fn = "lf_cross_attention_varlen";
  if (dtype != LF_DTYPE_BF16 && dtype != LF_DTYPE_F16)
    return set_error(LF_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or f16 only)", fn, dtype);
  if (head_dim <= 0 || head_dim > 128 || head_dim % 8 != 0)
    return set_error(LF_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 128)", fn, head_dim);
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0)
    return set_error(LF_ERR_INVALID, "%s: %d heads over %d key heads", fn, n_heads, n_kv_heads);
  if (n_q < 0 || n_kv < 0 || n_q > INT32_MAX - 128 || n_kv > INT32_MAX - 128 || n_items < 0 || max_q < 0 || max_kv < 0 ||
      total_kv < 0)
    return set_error(LF_ERR_INVALID, "%s: bad sizes", fn);
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(LF_ERR_INVALID, "%s: scale must be positive and finite", fn);
  if (n_items == 0 || n_q == 0 || max_q == 0) return LF_OK;
  if (q == nullptr || out == nullptr || items == nullptr || (n_kv > 0 && (k == nullptr || v == nullptr)))
    return set_error(LF_ERR_INVALID, "%s: null q, k, v, items or out", fn);
  const int64_t wq = int64_t(n_heads) * head_dim, wk = int64_t(n_kv_heads) * head_dim;
  if (ldq < wq || ld_out < wq || (n_kv > 0 && (ldk < wk || ldv < wk)))
    return set_error(LF_ERR_INVALID, "%s: a row stride is below its row", fn);
  if (!aligned16(q) || !aligned16(out) || !aligned16(items) || ldq % 8 || ld_out % 8 ||
      (n_kv > 0 && (!aligned16(k) || !aligned16(v) || ldk % 8 || ldv % 8)))
    return set_error(LF_ERR_INVALID, "%s: pointers and row strides must be 16-byte aligned", fn);
  CrossParams p;
  memset(&p, 0, sizeof(p));
  p.q = q;
  p.k = k;
  p.v = v;
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldv = ldv;
  p.n_q = n_q;
  p.n_kv = n_kv;
  p.n_heads = n_heads;
  p.n_kv_heads = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.d = head_dim;
  p.items = reinterpret_cast<const int4*>(items);
  p.n_items = n_items;
  p.max_q = max_q;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = out;
  p.ldo = ld_out;
  p.status = status;
  const int dev = current_device(), sms = device_sms(dev);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == LF_DTYPE_BF16;
  // Which kernel, and in how many parts the few-row kernel takes a sequence's keys: by their
  // times in us as measured on this GPU (launch aside), keys a sequence by their mean over the
  // records, the longest sequence from the start on (the records' order).
  // A few-row CTA takes 10.5 ns a key (64 columns; 13 at 128) alone and 20.5 with every place
  // taken (four or two an SM), between them by the square of the share taken, and 3 us beside
  // its keys, of which the first CTA's pass within the launch; clusters of four find nine
  // tenths of the places, of eight seven eighths.  Measured with the keys whole, in 2, 4 and 8
  // parts (64 columns, 16,384 keys each): 16 sequences x heads 172, 92, 51 and 33 us; 80: 174,
  // 102, 66 and 77; 192: 195, 128, 148 and 132; 320: 228, 275, 228 and 217; 512: 306, 316, 324
  // and 343; where 64 sequences of 20 to 10,668 keys, 935 on average, with 16 heads take 102 us
  // in eighths, 68 in quarters.
  // The other kernel takes 1.25 us a tile of 128 keys with one group of an SM at work, 2.0 with
  // two (64 keys at 128 columns: 0.95 and 1.05), and 2 us a unit.  Both, with launch, 16 heads
  // of 64: 8 sequences of 4,096 keys with 16 queries 32 and 50 us, 32: 46 and 50, 64: 79 and 50;
  // 1 of 8,192: 128 queries 46 and 87; 64 of 272: 32 queries 37 and 31; 200 of 100: 33 queries 82
  // and 43.
  const int64_t blocks = (int64_t(max_q) * p.group + kDecodeRows - 1) / kDecodeRows;
  const int64_t units = int64_t(n_items) * n_kv_heads;
  const int64_t mean_kv = total_kv / n_items < max_kv ? total_kv / n_items : max_kv;
  const bool narrow = head_dim <= 64;
  const double alone = narrow ? 0.0105 : 0.013, full = 0.0205, places = double(sms) * (narrow ? 4.0 : 2.0);
  int split = 1;
  double t_few = 0.0;
  for (int n = 1; n <= 8; n *= 2) {
    if (n > 1 && max_kv / n < 64) break;
    const double cap = places * (n <= 2 ? 1.0 : n == 4 ? 0.9 : 7.0 / 8.0);
    const double ctas = double(units) * double(blocks) * n, waves = std::floor(ctas / cap), rest = ctas / cap - waves;
    const double rate = alone + (full - alone) * std::fmin(1.0, ctas / cap * ctas / cap);  // of the first wave
    const double part = double(mean_kv) / n;
    const double last = rest > 0.0 ? part * (alone + (full - alone) * rest * rest) + 3.0 : 0.0;
    const double t = std::fmax(waves * (part * full + 3.0) + last, double(max_kv) / n * rate + 3.0);
    if (n == 1 || t < t_few) {
      t_few = t;
      split = n;
    }
  }
  const int64_t p_units = int64_t(n_items) * n_heads;
  const double p_keys = narrow ? 128.0 : 64.0, p_one = narrow ? 1.25 : 0.95, p_two = narrow ? 2.0 : 1.05;
  const double rounds = std::ceil(double(p_units) / (2.0 * sms));
  const double t_many = std::fmax(p_units <= sms ? 0.0 : rounds * (double(mean_kv) / p_keys * p_two + 2.0),
                                  std::ceil(double(max_kv) / p_keys) * p_one + 2.0);
  if (max_q <= kRows && t_few - 3.0 <= t_many && units * blocks * 8 <= INT32_MAX) {
    p.row_blocks = int32_t(blocks);
    p.split = split;
    if (narrow) return bf ? launch_decode<__nv_bfloat16, 64>(p, dev, s) : launch_decode<__half, 64>(p, dev, s);
    return bf ? launch_decode<__nv_bfloat16, 128>(p, dev, s) : launch_decode<__half, 128>(p, dev, s);
  }
  const int key_tile = narrow ? Shape<64>::kKeys : Shape<128>::kKeys;
  int rc;
  if ((rc = encode_rows(&p.q_map, dtype, q, ldq, n_q, n_heads, head_dim, kRows, "q"))) return rc;
  // no keys at all: the row read in the place of one (its result is not used) is a query row
  const void *kb = n_kv > 0 ? k : q, *vb = n_kv > 0 ? v : q;
  const int64_t kv_rows = n_kv > 0 ? n_kv : n_q;
  if ((rc = encode_rows(&p.k_map, dtype, kb, n_kv > 0 ? ldk : ldq, kv_rows, n_kv_heads, head_dim, key_tile, "k"))) return rc;
  if ((rc = encode_rows(&p.v_map, dtype, vb, n_kv > 0 ? ldv : ldq, kv_rows, n_kv_heads, head_dim, key_tile, "v"))) return rc;
  if (narrow) return bf ? launch_prompt<__nv_bfloat16, 64>(p, dev, s) : launch_prompt<__half, 64>(p, dev, s);
  return bf ? launch_prompt<__nv_bfloat16, 128>(p, dev, s) : launch_prompt<__half, 128>(p, dev, s);
}

extern "C" int lf_cross_attention_varlen(void* stream, int dtype, const void* q, int64_t ldq, int64_t n_q,
                                         const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t n_kv,
                                         int n_heads, int n_kv_heads, int head_dim, const int32_t* items, int n_items,
                                         int max_q, int max_kv, float scale, void* out, int64_t ld_out,
                                         int32_t* status) {
  return lf_cross_attention_varlen_total(stream, dtype, q, ldq, n_q, k, ldk, v, ldv, n_kv, n_heads, n_kv_heads, head_dim,
                                         items, n_items, max_q, max_kv, n_kv < 0 ? 0 : n_kv, scale, out, ld_out, status);
}
