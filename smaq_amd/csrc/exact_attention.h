// What the two attention kernels over exact keys share (not part of the C ABI).
#pragma once

#include <math.h>

#include "smaq_common.h"

namespace smaq {

constexpr float kLog2eF = 1.4426950408889634f;

// Scores in units of log2: scale, tanh cap and distance bias as the kernels apply
// them to a product q.k.
struct ScoreRule {
  float scale;  // no cap: scale log2(e); cap: 2 log2(e) scale / cap
  float cap;    // cap log2(e); 0: none
  int wide;     // the cap is above kWideCap
  float near;   // products below this in size may take near_score; 0: none
  float c[4];   // of near_score
};

// cap (1 - 2 / (e^(2x/cap) + 1)) loses what lies below some 2^-22 of the cap: up to
// this cap that moves a weight by less than 2^-13 (half a step of fp16 is 2^-11);
// above it small arguments take the series of tanh.
constexpr float kWideCap = 256.0f;

// tanh(y) / y as a polynomial in y^2: interpolated at Chebyshev's points for |y| <= kNearTanh,
// off by 2^-20.8 of the value at most, which is below 2^-21.9 of the cap.
constexpr double kNearTanh = 0.5;
constexpr double kTanh[4] = {0.99999945, -0.33326284, 0.13189939, -0.04439274};

// Whether rows of 16-bit elements start on 16 bytes.
template <typename... S>
inline bool rows_on_16(const void* p, S... strides) {
  return (uintptr_t)p % 16 == 0 && ((strides % 8 == 0) && ...);
}

// Whether the fp32 forms below hold: no scale or cap that leaves the range.
inline bool score_range(float scale, float cap) {
  return fabsf(scale) < 1e38f && (cap == 0.0f || (cap >= 1e-30f && cap < 1e30f));
}

inline ScoreRule score_rule(float scale, float cap) {
  if (cap > 0.0f) {
    // finite, so that a product of 0 has the score 0
    const double x = 2.0 * 1.4426950408889634 * (double)scale / (double)cap;
    ScoreRule r{(float)fmin(fmax(x, -3e38), 3e38), cap * kLog2eF, cap > kWideCap, 0.0f, {}};
    const double a = fabs((double)scale) / (double)cap, near = kNearTanh / a;
    bool fits = cap <= kWideCap && near > 1e-15 && near < 1e15;
    double f = 1.4426950408889634 * (double)scale;  // cap log2(e) a^(2k + 1)
    for (int k = 0; k < 4; ++k, f *= a * a) {
      r.c[k] = (float)(f * kTanh[k]);
      fits = fits && fabsf(r.c[k]) > 1e-37f && fabsf(r.c[k]) < 1e37f;
    }
    if (fits) r.near = (float)near;
    return r;
  }
  return {scale * kLog2eF, 0.0f, 0, 0.0f, {}};
}

// cap tanh(x / cap) of x = scale dot, times log2(e).  The limits at +-inf are exact,
// NaN passes.
template <bool WIDE>
__device__ __forceinline__ float capped_score(const ScoreRule& r, float dot) {
  const float x = dot * r.scale;
  const float t = fmaf(-2.0f * r.cap, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x) + 1.0f), r.cap);
  if constexpr (!WIDE) return t;
  // y = x / (2 log2 e): y - y^3/3 + 2 y^5/15 - 17 y^7/315 + 62 y^9/2835, below 0.35 to 2^-21
  const float y = x * (0.5f / kLog2eF), z = y * y;
  const float s = fmaf(z, fmaf(z, fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f);
  return fabsf(y) < 0.35f ? r.cap * fmaf(y * z, s, y) : t;
}

// The same for |dot| < near, with no exponential or reciprocal: 16384 capped tokens 2.69 ->
// 2.59 ms, 256 dims 1.04 -> 0.91.
__device__ __forceinline__ float near_score(const ScoreRule& r, float dot, float less = 0.0f) {
  const float z = dot * dot;
  return fmaf(dot, fmaf(z, fmaf(z, fmaf(z, r.c[3], r.c[2]), r.c[1]), r.c[0]), -less);
}

// put(i, score of the product get(i)) for N products: one uniform choice of the rule
template <int N, typename Get, typename Put>
__device__ __forceinline__ void each_score(const ScoreRule& r, Get get, Put put) {
  if (r.cap == 0.0f) {
#pragma unroll
    for (int i = 0; i < N; ++i) put(i, get(i) * r.scale);
  } else if (!r.wide) {
#pragma unroll
    for (int i = 0; i < N; ++i) put(i, capped_score<false>(r, get(i)));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) put(i, capped_score<true>(r, get(i)));
  }
}

// ------------------------------------------------------- matrix operands ---
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

template <typename T>
struct Mat;

template <>
struct Mat<_Float16> {
  static constexpr uint32_t kExp = 0x7c00;  // exponent bits
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4v mma16(u32x4v a, u32x4v b, f32x4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16v mma32(u32x4v a, u32x4v b, f32x16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  // two numbers rounded to nearest, packed
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){x, y}, v2));
  }
};

template <>
struct Mat<bf16> {
  static constexpr uint32_t kExp = 0x7f80;
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4v mma16(u32x4v a, u32x4v b, f32x4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16v mma32(u32x4v a, u32x4v b, f32x16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){x, y}, v2));
  }
};

// ones over the halves of a word of two numbers that are infinite or NaN
template <uint32_t EXP>
__device__ __forceinline__ uint32_t not_finite_halves(uint32_t w) {
  return ((w & EXP) == EXP ? 0xffffu : 0u) | ((w & (EXP << 16)) == (EXP << 16) ? 0xffff0000u : 0u);
}

// 16-bit halves of two words: (low x, low y) or (high x, high y)
__device__ __forceinline__ uint32_t low_halves(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07060302u); }

constexpr float kNegInf = -__builtin_inff();
// A softmax's reference maximum is raised when a score is this much (log2) above it:
// weights stay below 2^8, far inside fp16, and sums and outputs are rarely rescaled.
constexpr float kRaise = 8.0f;

}  // namespace smaq
