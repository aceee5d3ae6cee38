// Rotary positions: of a row's first r dims the pairs (a, b) = (x_i, x_{i + r/2}), or
// interleaved (x_{2i}, x_{2i+1}), are turned by the angle of the token's position,
//   a' = a cos - b sin,   b' = b cos + a sin,
// with cos and sin from a table [tokens][r/2][2] in fp64 that is made once a step.
//
// The products are in fp64: a row of the 4-bit cache is quantized after it is turned, and its
// codes then follow from the inputs alone, whichever kernel turned them and in which order.  That
// costs nothing where it counts: the rows come from memory at a rate that leaves the fp64 units
// idle most of the time.  2047 tokens, 32 heads of 80 dims: 9.2 us, 2.3 TB/s of rows that lie in the caches;
// one token 2.5 us, a launch and two loads one after the other.
#pragma once
#include "kv4_device.h"

namespace rotary {

using kv4::u32x4;

typedef double double2_t __attribute__((ext_vector_type(2)));  // cos, sin

// The turned value, rounded to fp32 on the way to the row's type as every value is.  (The compiler
// must not see both roundings: it makes one of them, in 40 operations, in some kernels and not in
// others.)
__device__ __forceinline__ float rounded(double x) {
  float y = (float)x;
  asm("" : "+v"(y));
  return y;
}
__device__ __forceinline__ float first_of(double a, double b, double2_t t) {
  return rounded(__builtin_fma(-b, t.y, a * t.x));
}
__device__ __forceinline__ float second_of(double a, double b, double2_t t) {
  return rounded(__builtin_fma(a, t.y, b * t.x));
}

struct Rows {
  const uint16_t* x;
  uint16_t* y;
  const double2_t* angles;    // [tokens][pairs]
  long long xt, xh, yt, yh;   // strides in elements
  int tokens, heads, head_dim, pairs;
};

// Whether units of eight pairs (and of eight other dims) are whole 16-byte pieces.
__host__ __device__ inline bool aligned(int pairs, bool interleaved) {
  return pairs % (interleaved ? 4 : 8) == 0;
}
// Units of a row: of eight pairs (interleaved and aligned: of four, which lie together), then of
// eight dims that are not turned.
__host__ __device__ inline int turning_units(int pairs, bool interleaved) {
  return interleaved && aligned(pairs, true) ? pairs / 4 : (pairs + 7) / 8;
}
__host__ __device__ inline int units(int head_dim, int pairs, bool interleaved) {
  return turning_units(pairs, interleaved) + (head_dim - 2 * pairs + 7) / 8;
}

constexpr int kThreads = 256;

// How a workgroup's threads share out rows: `heads` of `tokens` at a time, a unit a thread.
struct Shape {
  int units, heads, tokens;
};
__host__ __device__ inline Shape shape_of(int head_dim, int pairs, bool interleaved, int heads) {
  Shape s;
  s.units = units(head_dim, pairs, interleaved);
  const int slots = kThreads / s.units;  // (units <= 128 / ... checked on the host)
  s.heads = heads < slots ? heads : slots;
  s.tokens = slots / s.heads;
  return s;
}

// One workgroup's rows: tokens [token0, + s.tokens) and heads head0, head0 + s.heads, ... below head_end.
// A thread owns both values of its pairs, so y may be x.
template <int TYPE, bool INTERLEAVED, bool ALIGNED>
__device__ __forceinline__ void turn_rows(const Rows& a, const Shape& s, int token0, int head0, int head_end) {
  const int tid = threadIdx.x;
  const int slot = tid / s.units, u = tid - slot * s.units;
  const int t = slot / s.heads, token = token0 + t;
  if (t >= s.tokens || token >= a.tokens) return;
  const int turning = turning_units(a.pairs, INTERLEAVED), r = 2 * a.pairs;
  const uint16_t* x = a.x + token * a.xt;
  uint16_t* y = a.y + token * a.yt;
  const double2_t* at = a.angles + (size_t)token * a.pairs;
  const int head = head0 + slot - t * s.heads;
  if (u >= turning) {  // dims that stay
    if (a.x == a.y) return;
    const int d = r + 8 * (u - turning);
    for (int h = head; h < head_end; h += s.heads) {
      if constexpr (ALIGNED) {
        *reinterpret_cast<u32x4*>(y + h * a.yh + d) = *reinterpret_cast<const u32x4*>(x + h * a.xh + d);
      } else {
        for (int i = 0; i < 8 && d + i < a.head_dim; i++) y[h * a.yh + d + i] = x[h * a.xh + d + i];
      }
    }
    return;
  }
  if constexpr (ALIGNED && INTERLEAVED) {
    double2_t cs[4];
#pragma unroll
    for (int i = 0; i < 4; i++) cs[i] = at[4 * u + i];
    for (int h = head; h < head_end; h += s.heads) {
      float v[8];
      kv4::unpack8<TYPE>(*reinterpret_cast<const u32x4*>(x + h * a.xh + 8 * u), v);
      float o[8];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        o[2 * i] = first_of(v[2 * i], v[2 * i + 1], cs[i]);
        o[2 * i + 1] = second_of(v[2 * i], v[2 * i + 1], cs[i]);
      }
      *reinterpret_cast<u32x4*>(y + h * a.yh + 8 * u) = kv4::pack8<TYPE>(o);
    }
  } else if constexpr (ALIGNED) {
    double2_t cs[8];
#pragma unroll
    for (int i = 0; i < 8; i++) cs[i] = at[8 * u + i];
    for (int h = head; h < head_end; h += s.heads) {
      float lo[8], hi[8], p[8], q[8];
      kv4::unpack8<TYPE>(*reinterpret_cast<const u32x4*>(x + h * a.xh + 8 * u), lo);
      kv4::unpack8<TYPE>(*reinterpret_cast<const u32x4*>(x + h * a.xh + a.pairs + 8 * u), hi);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        p[i] = first_of(lo[i], hi[i], cs[i]);
        q[i] = second_of(lo[i], hi[i], cs[i]);
      }
      *reinterpret_cast<u32x4*>(y + h * a.yh + 8 * u) = kv4::pack8<TYPE>(p);
      *reinterpret_cast<u32x4*>(y + h * a.yh + a.pairs + 8 * u) = kv4::pack8<TYPE>(q);
    }
  } else {
    for (int h = head; h < head_end; h += s.heads) {
      for (int i = 8 * u; i < min(8 * u + 8, a.pairs); i++) {
        const int lo = INTERLEAVED ? 2 * i : i, hi = INTERLEAVED ? 2 * i + 1 : i + a.pairs;
        const double p = kv4::to_float<TYPE>(x[h * a.xh + lo]), q = kv4::to_float<TYPE>(x[h * a.xh + hi]);
        const double2_t cs = at[i];
        y[h * a.yh + lo] = kv4::from_float<TYPE>(first_of(p, q, cs));
        y[h * a.yh + hi] = kv4::from_float<TYPE>(second_of(p, q, cs));
      }
    }
  }
}

// Eight dims [8 b, 8 b + 8) of a row, turned and rounded to the row's type.  `raw` are those dims.
template <int TYPE, bool INTERLEAVED, bool ALIGNED>
struct Turn {
  double2_t cs[INTERLEAVED ? 4 : 8];
  int partner;  // first of the dims that the eight are paired with (half layout)
  int kind;     // 0: they stay, 1: firsts of their pairs, 2: seconds

  __device__ __forceinline__ Turn(const double2_t* at, int pairs, int b) {
    if constexpr (!ALIGNED) return;
    const int d = 8 * b;
    kind = d >= 2 * pairs ? 0 : INTERLEAVED || d < pairs ? 1 : 2;
    partner = kind == 2 ? d - pairs : d + pairs;
    const int first = INTERLEAVED ? d / 2 : kind == 2 ? d - pairs : d;
#pragma unroll
    for (int i = 0; i < (INTERLEAVED ? 4 : 8); i++) cs[i] = kind == 0 ? (double2_t){1., 0.} : at[first + i];
  }

  __device__ __forceinline__ u32x4 operator()(const u32x4& raw, const uint16_t* row, const double2_t* at, int pairs,
                                              int b) const {
    float v[8], o[8];
    kv4::unpack8<TYPE>(raw, v);
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int d = 8 * b + i;
        o[i] = v[i];
        if (d >= 2 * pairs) continue;
        const bool first = INTERLEAVED ? d % 2 == 0 : d < pairs;
        const int pair = INTERLEAVED ? d / 2 : first ? d : d - pairs;
        const double w = kv4::to_float<TYPE>(row[INTERLEAVED ? d ^ 1 : first ? d + pairs : d - pairs]);
        o[i] = first ? first_of(v[i], w, at[pair]) : second_of(w, v[i], at[pair]);
      }
      return kv4::pack8<TYPE>(o);
    } else if constexpr (INTERLEAVED) {
      if (kind == 0) return raw;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        o[2 * i] = first_of(v[2 * i], v[2 * i + 1], cs[i]);
        o[2 * i + 1] = second_of(v[2 * i], v[2 * i + 1], cs[i]);
      }
      return kv4::pack8<TYPE>(o);
    } else {
      if (kind == 0) return raw;
      float w[8];
      kv4::unpack8<TYPE>(*reinterpret_cast<const u32x4*>(row + partner), w);
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = kind == 1 ? first_of(v[i], w[i], cs[i]) : second_of(w[i], v[i], cs[i]);
      return kv4::pack8<TYPE>(o);
    }
  }
};

// f(bool_constant<INTERLEAVED>, bool_constant<ALIGNED>)
template <class F>
void dispatch(int pairs, bool interleaved, F&& f) {
  const bool al = aligned(pairs, interleaved);
  if (interleaved) al ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
  else al ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}

}  // namespace rotary
