// Symmetric 8-bit quantisation of a row: with top = max |x| over the row,
//     scale = top / 127                 (rounded to f32)
//     q     = round_half_even(127 x / top)          in [-127, 127]
// The quotient is decided exactly.  For f32 rows it is formed as v = x * (127 / top), which
// is off by at most 127.5 * 2^-23 < 2^-15, and where v lies nearer than 2^-15 to a half the
// remainder decides (quant_settle).  With 16-bit values exact halves are frequent (0.5% of
// bf16's: one or more in most warps' 32), so their quotients are divided out instead
// (RowQuant::q8): v = v0 + (p - v0 top) / top with p = 127 x and v0 = p * (1 / top), where
// the FMA makes p - v0 top exact, is the quotient itself whenever f32 holds it, as it
// holds every half; and a quotient of two values of at most 11 bits that is not a half is
// 2^(k - 12) or more away from one (k the exponent of x less that of top) where v is
// 2^(k - 16) off.  So q does not depend on how a caller rounds, and ties go to the even
// step.  A row of zeros gives q = 0, scale = 0.  A row with an infinity or
// NaN gives q = 0 and scale = NaN, so that whatever is computed from the row is NaN.
#pragma once

#include "lf_common.cuh"

namespace lf {

// |x| as an integer that orders like the magnitude, NaN above infinity (fmaxf would drop NaN).
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Rounds 127 x / top where v = x * (127 / top) lies next to r + 1/2 or r - 1/2 (r = rint(v)),
// or is not a number: 127 x - r top is exact in two floats (the product 127 x splits
// exactly, and its head minus r top is a multiple of ulp(top) / 2 below 2^24 of them), so
// comparing it with top / 2 is exact.  Rare, and out of line: inlined for each of a lane's
// 32 values it doubled the kernels' code and time.
__device__ __noinline__ static float quant_settle(float x, float r, float top, float inv) {
  if (!(fabsf(r) <= 128.f) || inv == 0.f) return 0.f;  // only rows that are not finite (or all 0) come here so
  const float p = 127.f * x, e = fmaf(127.f, x, -p), rem = fmaf(-r, top, p);
  const float sgn = rem < 0.f ? -1.f : 1.f;
  const float over = (fabsf(rem) - 0.5f * top) + sgn * e;  // its sign is exact: the difference is
  const bool odd = (int(r) & 1) != 0;
  return over > 0.f || (over == 0.f && odd) ? r + sgn : r;
}

struct RowQuant {
  static constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, ties to even
  float pre;    // a power of two that keeps top and 127 x clear of f32's ends
  float top;    // the row's largest magnitude, times pre
  float inv;    // 127 / top; 0 for a row of zeros or a row that is not finite
  float scale;
  float raw;      // the row's largest magnitude where it is well inside f32's range; else 0
  float rcp;      // 1 / raw, inv_raw = 127 / raw (0 where raw is)
  float inv_raw;
  // top_bits: the largest mag_bits of the row
  __device__ __forceinline__ explicit RowQuant(uint32_t top_bits) {
    const float t = __uint_as_float(top_bits);
    const bool finite = top_bits < 0x7f800000u;
    pre = t < 1.f ? 18446744073709551616.f : 1.f / 18446744073709551616.f;
    top = t * pre;
    inv = (top_bits == 0u || !finite) ? 0.f : __fdiv_rn(127.f, top);
    scale = finite ? __fdiv_rn(t, 127.f) : __uint_as_float(0x7fc00000u);
    raw = t > 0x1p-100f && t < 0x1p100f ? t : 0.f;  // NaN and infinity: 0
    rcp = raw != 0.f ? __frcp_rn(raw) : 0.f;
    inv_raw = raw != 0.f ? __fdiv_rn(127.f, raw) : 0.f;
  }
  // q in the low byte (two's complement) of the result
  __device__ __forceinline__ uint32_t q(float x) const {
    x *= pre;
    const float v = x * inv;
    float m = v + kMagic;
    const float r = m - kMagic;
    if (!(fabsf(v - r) < 0.499969482421875f)) m = quant_settle(x, r, top, inv) + kMagic;
    return __float_as_uint(m);
  }
  // q of four values, the first in the low byte
  __device__ __forceinline__ uint32_t q4(float a, float b, float c, float d) const {
    return __byte_perm(__byte_perm(q(a), q(b), 0x0040), __byte_perm(q(c), q(d), 0x0040), 0x5410);
  }
  // q of eight values of type T, the first in the low byte of x.  Rows at the ends of f32's
  // range take q4, and of f32 rows any eight with a value next to a half.
  template <typename T>
  __device__ __forceinline__ uint2 q8(const float (&x)[8]) const {
    uint32_t m[8];
    bool slow = raw == 0.f;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = f2_mul(make_float2(x[2 * i], x[2 * i + 1]), f2(127.f));
        const float2 v0 = f2_mul(p, f2(rcp));
        const float2 v = f2_fma(f2_fma(v0, f2(-raw), p), f2(rcp), v0);
        const float2 w = f2_add(v, f2(kMagic));
        m[2 * i] = __float_as_uint(w.x);
        m[2 * i + 1] = __float_as_uint(w.y);
      }
    } else {
      float far = 0.f;  // the largest distance to the nearest integer
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = f2_mul(make_float2(x[2 * i], x[2 * i + 1]), f2(inv_raw));
        const float2 w = f2_add(v, f2(kMagic));
        const float2 d = f2_add(v, f2_fma(w, f2(-1.f), f2(kMagic)));  // v - (w - magic), both exact
        far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
        m[2 * i] = __float_as_uint(w.x);
        m[2 * i + 1] = __float_as_uint(w.y);
      }
      slow |= far >= 0.499969482421875f;
    }
    if (slow) return make_uint2(q4(x[0], x[1], x[2], x[3]), q4(x[4], x[5], x[6], x[7]));
    return make_uint2(
        __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410),
        __byte_perm(__byte_perm(m[4], m[5], 0x0040), __byte_perm(m[6], m[7], 0x0040), 0x5410));
  }
};

// A lane's 8 elements of a 256-element chunk: neighbours (VEC), kept as they lie in memory
// until they are rounded, or 32 apart.  Elements past the row read as 0.
template <typename T, bool VEC>
struct QuantChunk {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* row, int32_t base, int lane, int32_t cols) {
    if constexpr (VEC) {
      const int32_t col = base + lane * 8;
#pragma unroll
      for (int i = 0; i < int(sizeof(T)) / 2; ++i)
        w[i] = col < cols ? __ldg(reinterpret_cast<const uint4*>(row + col) + i) : make_uint4(0u, 0u, 0u, 0u);
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int32_t col = base + i * 32 + lane;
        e[i] = col < cols ? row[col] : DT<T>::from_f(0.f);
      }
#pragma unroll
      for (int i = 0; i < int(sizeof(T)) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  }
  // VEC's elements of a 16-bit row of any alignment: pairs where they are aligned, and the two
  // single elements around them where the row starts between pairs.
  __device__ __forceinline__ void load_near(const T* row, int32_t base, int lane, int32_t cols) {
    static_assert(VEC && sizeof(T) == 2, "16-bit neighbours");
    const int32_t col = base + lane * 8;
    const uint16_t* at = reinterpret_cast<const uint16_t*>(row + col);
    uint32_t u[4] = {0u, 0u, 0u, 0u};
    if (col + 8 <= cols) {
      if ((reinterpret_cast<uintptr_t>(row) & 2u) == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
      } else {
        const uint32_t first = __ldg(at), last = __ldg(at + 7);
        uint32_t m[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) m[i] = __ldg(reinterpret_cast<const uint32_t*>(at + 1) + i);
        u[0] = first | (m[0] << 16);
        u[1] = __funnelshift_r(m[0], m[1], 16);
        u[2] = __funnelshift_r(m[1], m[2], 16);
        u[3] = (m[2] >> 16) | (last << 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < cols) u[i >> 1] |= uint32_t(__ldg(at + i)) << (16 * (i & 1));
    }
    w[0] = make_uint4(u[0], u[1], u[2], u[3]);
  }
  // eight values, rounded to T
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i) {
      if constexpr (sizeof(T) == 2)
        w[i] = make_uint4(Pack2<T>::pack(v[0], v[1]), Pack2<T>::pack(v[2], v[3]), Pack2<T>::pack(v[4], v[5]),
                          Pack2<T>::pack(v[6], v[7]));
      else
        w[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                          __float_as_uint(v[4 * i + 3]));
    }
  }
  // the largest magnitude as an integer that orders like it: two 16-bit halves, or 32 bits
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 2) t = __vmaxu2(t, u[k] & 0x7fff7fffu);
        else t = max(t, u[k] & 0x7fffffffu);
      }
    }
    return t;
  }
  // the eight steps, the lane's first element in the low byte of x
  __device__ __forceinline__ uint2 steps(const RowQuant& rq) const {
    float v[8];
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 2) {
          const float2 f = Pack2<T>::unpack(u[k]);
          v[2 * k] = f.x;
          v[2 * k + 1] = f.y;
        } else {
          v[4 * i + k] = __uint_as_float(u[k]);
        }
      }
    }
    return rq.template q8<T>(v);
  }
  __device__ __forceinline__ void store(int8_t* row, int32_t base, int lane, int32_t cols, const RowQuant& rq) const {
    const uint2 q = steps(rq);
    if constexpr (VEC) {
      const int32_t col = base + lane * 8;
      if (col + 8 <= cols) {
        *reinterpret_cast<uint2*>(row + col) = q;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < cols) row[col + i] = int8_t((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xffu);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int32_t col = base + i * 32 + lane;
        if (col < cols) row[col] = int8_t((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xffu);
      }
    }
  }
};

// The f32 bits of a magnitude given by its type's bits.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t t) {
  if constexpr (sizeof(T) == 2) {
    const uint16_t h = uint16_t(t);
    return __float_as_uint(DT<T>::to_f(*reinterpret_cast<const T*>(&h)));
  }
  return t;
}

}  // namespace lf
