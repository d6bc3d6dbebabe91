// Arithmetic of the dense operators: the activations with their derivatives, the 8-bit form of kept activations, packing.
#pragma once

#include "tab_common.cuh"

namespace tab {

// ---- activations ---------------------------------------------------------------------------------------------------------
// fp32 throughout.  silu and the tanh form of GELU are both z * sigmoid(u): 0.5 (1 + tanh v) = 1 / (1 + exp(-2 v)), which
// needs no cancelling sum for very negative z.

__device__ __forceinline__ float sigmoid_f(float u) { return __fdividef(1.0f, 1.0f + __expf(-u)); }

constexpr float kGeluC = 0.7978845608028654f;      // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;
constexpr float kInvSqrt2 = 0.7071067811865476f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

// Normal distribution function c = (1 + erf(z / sqrt 2)) / 2 and e = exp(-z^2 / 2), by Abramowitz and Stegun 7.1.26: with
// x = |z| / sqrt 2 and t = 1 / (1 + 0.3275911 x), erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2) within 1.5e-7.  The exponential serves
// the derivative as well; erff takes about twice the instructions and a branch.
__device__ __forceinline__ void normal_cdf(float z, float& c, float& e) {
  const float t = __fdividef(1.0f, __fmaf_rn(0.3275911f * kInvSqrt2, fabsf(z), 1.0f));
  e = __expf(-0.5f * z * z);
  float q = __fmaf_rn(1.061405429f, t, -1.453152027f);
  q = __fmaf_rn(q, t, 1.421413741f);
  q = __fmaf_rn(q, t, -0.284496736f);
  q = __fmaf_rn(q, t, 0.254829592f);
  const float tail = 0.5f * q * t * e;             // the side away from zero
  c = z < 0.f ? tail : 1.0f - tail;
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == TAB_ACT_RELU) return z < 0.f ? 0.f : z;     // NaN stays NaN
  if constexpr (ACT == TAB_ACT_SILU) return z * sigmoid_f(z);
  if constexpr (ACT == TAB_ACT_GELU) {
    float c, e;
    normal_cdf(z, c, e);
    return z * c;
  }
  if constexpr (ACT == TAB_ACT_GELU_TANH) return z * sigmoid_f(2.0f * kGeluC * z * (1.0f + kGeluA * z * z));
  return z;
}

// value and derivative
template <int ACT>
__device__ __forceinline__ void act_both(float z, float& a, float& d) {
  if constexpr (ACT == TAB_ACT_RELU) {
    a = z < 0.f ? 0.f : z;
    d = z <= 0.f ? 0.f : z > 0.f ? 1.f : z;                          // in the derivative too
  } else if constexpr (ACT == TAB_ACT_SILU) {
    const float s = sigmoid_f(z);
    a = z * s;
    d = s * (1.0f + z * (1.0f - s));
  } else if constexpr (ACT == TAB_ACT_GELU) {
    float c, e;
    normal_cdf(z, c, e);
    a = z * c;
    d = c + z * kInvSqrt2Pi * e;
  } else if constexpr (ACT == TAB_ACT_GELU_TANH) {
    const float s = sigmoid_f(2.0f * kGeluC * z * (1.0f + kGeluA * z * z));
    a = z * s;
    d = s + z * s * (1.0f - s) * (2.0f * kGeluC * (1.0f + 3.0f * kGeluA * z * z));
  } else {
    a = z;
    d = 1.f;
  }
}

template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};

// Calls f(ActTag<act>()): the choice is made once per chunk of values, outside the loops over them.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case TAB_ACT_RELU: f(ActTag<TAB_ACT_RELU>()); break;
    case TAB_ACT_SILU: f(ActTag<TAB_ACT_SILU>()); break;
    case TAB_ACT_GELU: f(ActTag<TAB_ACT_GELU>()); break;
    case TAB_ACT_GELU_TANH: f(ActTag<TAB_ACT_GELU_TANH>()); break;
    default: f(ActTag<TAB_ACT_NONE>()); break;
  }
}

// ---- 8-bit blocks --------------------------------------------------------------------------------------------------------
// 64 values of a row share a scale: scale = amax / 127, q = rint(v / scale).  A block that holds a value that is not
// finite is kept as q = 0 with the scale NaN, so that it comes back as NaN and an overflow is not lost on the way.
constexpr int kKeepBlock = 64;

__device__ __forceinline__ RowQuant make_block_quant(float amax, bool finite) {
  RowQuant rq = make_row_quant_fast(amax);
  if (!finite) {
    rq.scale = __int_as_float(0x7fc00000);
    rq.inv = 0.f;
    rq.exact = false;
  }
  return rq;                         // quant8 gives zeros where !(scale > 0): NaN included
}

// Two fp32 operations in one instruction, each rounded as the single one is.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// quant8 (the correctly rounded quotient, rounded half to even, in the low bytes) on pairs of values.
__device__ __forceinline__ uint2 block_quant8(const float (&v)[8], const RowQuant& rq) {
  if (rq.exact || !(rq.scale > 0.f)) return quant8(v, rq);
  const uint64_t inv = f32x2(rq.inv, rq.inv), minus_scale = f32x2(-rq.scale, -rq.scale), magic = f32x2(kRoundMagic, kRoundMagic);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t x = f32x2(v[2 * i], v[2 * i + 1]);
    const uint64_t q0 = mul_f32x2(x, inv);
    const uint64_t q1 = fma_f32x2(fma_f32x2(q0, minus_scale, x), inv, q0);
    const uint64_t r = add_f32x2(q1, magic);
    w[2 * i] = static_cast<uint32_t>(r);
    w[2 * i + 1] = static_cast<uint32_t>(r >> 32);
  }
  return make_uint2(pack4_words(w[0], w[1], w[2], w[3]), pack4_words(w[4], w[5], w[6], w[7]));
}

// ---- packing -------------------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 8 values of a row of n that may begin and end anywhere, columns >= n as zero
template <typename T>
__device__ __forceinline__ void load8_any(const T* row, int col, int n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = col + i < n ? Elem<T>::to_f32(row[col + i]) : 0.f;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

}  // namespace tab
