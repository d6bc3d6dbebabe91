// Arithmetic of the dense operators: the activations with their derivatives, the 8-bit form of kept activations, packing.
#pragma once

#include "tab_common.cuh"

namespace tab {

// Two fp32 operations in one instruction, each rounded as the single one is.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 from_f32x2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
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
__device__ __forceinline__ uint64_t splat(float a) { return f32x2(a, a); }

// ---- activations ---------------------------------------------------------------------------------------------------------
// fp32 throughout, on pairs of values: the exponential and the reciprocal are the hardware's (2 and 1 units in the last place), all
// else is two values to an instruction.  What they cost is instructions: 8192 x 7168 values of the GELU derivative from and to HBM
// took 73 us one by one, 60 so (bytes: 54).  silu and the tanh form of GELU are both z * sigmoid(u): 0.5 (1 + tanh v) = 1 / (1 + exp(-2 v)),
// which needs no cancelling sum for very negative z.
__device__ __forceinline__ uint64_t exp2_f32x2(uint64_t v) {
  float2 f = from_f32x2(v);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.y));
  return f32x2(f.x, f.y);
}
__device__ __forceinline__ uint64_t rcp_f32x2(uint64_t v) {
  float2 f = from_f32x2(v);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.y));
  return f32x2(f.x, f.y);
}

constexpr float kGeluC = 0.7978845608028654f;      // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;
constexpr float kInvSqrt2 = 0.7071067811865476f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

// 1 / (1 + 2^u)
__device__ __forceinline__ uint64_t logistic2(uint64_t u) { return rcp_f32x2(add_f32x2(exp2_f32x2(u), splat(1.f))); }

// Normal distribution function c = (1 + erf(z / sqrt 2)) / 2 and e = exp(-z^2 / 2), by Abramowitz and Stegun 7.1.26: with
// x = |z| / sqrt 2 and t = 1 / (1 + 0.3275911 x), erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2) within 1.5e-7.  The exponential serves
// the derivative as well; erff takes about twice the instructions and a branch.  GELU is within 2.1e-7 of its value everywhere; relative
// to the value that is 5e-5 at z = -3, 5e-4 at -4 (half an fp16 step there), 1.6e-3 at -5, 3.6e-3 at -6 (half a bf16 step) and 1e-2 at -8.
// 1 + erff is closer down to about -4.5 and cancels below: 4e-2 off at -5, nothing left at -6.
__device__ __forceinline__ void normal_cdf(uint64_t z, uint64_t& c, uint64_t& e) {
  const float2 f = from_f32x2(z);
  const uint64_t t = rcp_f32x2(fma_f32x2(f32x2(fabsf(f.x), fabsf(f.y)), splat(0.3275911f * kInvSqrt2), splat(1.f)));
  e = exp2_f32x2(mul_f32x2(mul_f32x2(z, z), splat(-0.5f * kLog2e)));
  uint64_t q = fma_f32x2(t, splat(0.5f * 1.061405429f), splat(0.5f * -1.453152027f));
  q = fma_f32x2(q, t, splat(0.5f * 1.421413741f));
  q = fma_f32x2(q, t, splat(0.5f * -0.284496736f));
  q = fma_f32x2(q, t, splat(0.5f * 0.254829592f));
  const uint64_t tail = mul_f32x2(mul_f32x2(q, t), e);             // the side away from zero
  const float2 near = from_f32x2(fma_f32x2(tail, splat(-1.f), splat(1.f))), far = from_f32x2(tail);
  c = f32x2(f.x < 0.f ? far.x : near.x, f.y < 0.f ? far.y : near.y);
}

// a = act(z), d = act'(z); what a caller does not use is not computed
template <int ACT>
__device__ __forceinline__ void act_pair(uint64_t z, uint64_t& a, uint64_t& d) {
  const uint64_t one = splat(1.f), minus = splat(-1.f);
  if constexpr (ACT == TAB_ACT_RELU) {
    const float2 f = from_f32x2(z);
    a = f32x2(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);       // NaN stays NaN, in the derivative too
    d = f32x2(f.x <= 0.f ? 0.f : f.x > 0.f ? 1.f : f.x, f.y <= 0.f ? 0.f : f.y > 0.f ? 1.f : f.y);
  } else if constexpr (ACT == TAB_ACT_SILU) {
    const uint64_t s = logistic2(mul_f32x2(z, splat(-kLog2e)));
    a = mul_f32x2(z, s);
    d = mul_f32x2(s, fma_f32x2(z, fma_f32x2(s, minus, one), one));                 // s (1 + z (1 - s))
  } else if constexpr (ACT == TAB_ACT_GELU) {
    uint64_t c, e;
    normal_cdf(z, c, e);
    a = mul_f32x2(z, c);
    d = fma_f32x2(mul_f32x2(z, splat(kInvSqrt2Pi)), e, c);
  } else if constexpr (ACT == TAB_ACT_GELU_TANH) {
    const uint64_t zz = mul_f32x2(z, z);
    const uint64_t s = logistic2(mul_f32x2(z, fma_f32x2(zz, splat(-2.f * kLog2e * kGeluC * kGeluA), splat(-2.f * kLog2e * kGeluC))));
    a = mul_f32x2(z, s);
    // s + z s (1 - s) 2 C (1 + 3 A z^2)
    d = fma_f32x2(mul_f32x2(a, fma_f32x2(s, minus, one)), fma_f32x2(zz, splat(6.f * kGeluC * kGeluA), splat(2.f * kGeluC)), s);
  } else {
    a = z;
    d = one;
  }
}

// v[i] = act(v[i])
template <int ACT, int N>
__device__ __forceinline__ void act_values(float (&v)[N]) {
  if constexpr (ACT == TAB_ACT_NONE) return;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    uint64_t a, d;
    act_pair<ACT>(f32x2(v[i], v[i + 1]), a, d);
    const float2 f = from_f32x2(a);
    v[i] = f.x;
    v[i + 1] = f.y;
  }
}

// g[i] = act(g[i]) u[i]
template <int ACT, int N>
__device__ __forceinline__ void act_gate(float (&g)[N], const float (&u)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    uint64_t a, d;
    act_pair<ACT>(f32x2(g[i], g[i + 1]), a, d);
    const float2 f = from_f32x2(mul_f32x2(a, f32x2(u[i], u[i + 1])));
    g[i] = f.x;
    g[i + 1] = f.y;
  }
}

// the same backwards: g, u, dh = gate, up values and d(act(gate) up) become d(gate) = dh u act'(gate), d(up) = dh act(gate) and act(gate) u
template <int ACT, int N>
__device__ __forceinline__ void act_gate_grad(float (&g)[N], float (&u)[N], float (&dh)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t up = f32x2(u[i], u[i + 1]), grad = f32x2(dh[i], dh[i + 1]);
    uint64_t a, d;
    act_pair<ACT>(f32x2(g[i], g[i + 1]), a, d);
    const float2 dg = from_f32x2(mul_f32x2(mul_f32x2(grad, up), d)), du = from_f32x2(mul_f32x2(grad, a)), h = from_f32x2(mul_f32x2(a, up));
    g[i] = dg.x;
    g[i + 1] = dg.y;
    u[i] = du.x;
    u[i + 1] = du.y;
    dh[i] = h.x;
    dh[i + 1] = h.y;
  }
}

// g[i] *= act'(z[i])
template <int ACT, int N>
__device__ __forceinline__ void act_slope(float (&g)[N], const float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    uint64_t a, d;
    act_pair<ACT>(f32x2(z[i], z[i + 1]), a, d);
    const float2 f = from_f32x2(mul_f32x2(f32x2(g[i], g[i + 1]), d));
    g[i] = f.x;
    g[i + 1] = f.y;
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
