// dense_math.cuh - element arithmetic of the dense feed-forward operators: 16-bit conversions, activations and their slopes.
#pragma once

#include "common.cuh"
#include "dense.hpp"

namespace vkernels::kernels::cuda {

namespace {

template <int TYPE>
__device__ __forceinline__ float dense_to_f32(uint16_t v) {
  if constexpr (TYPE == kDenseBf16) return __uint_as_float((uint32_t)v << 16);
  return __half2float(__ushort_as_half(v));
}
template <int TYPE>
__device__ __forceinline__ uint16_t dense_from_f32(float v) {
  if constexpr (TYPE == kDenseBf16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}
template <int TYPE>
__device__ __forceinline__ uint32_t dense_pack(float lo, float hi) {
  if constexpr (TYPE == kDenseBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int TYPE>
__device__ __forceinline__ float2 dense_unpack(uint32_t v) {
  return make_float2(dense_to_f32<TYPE>((uint16_t)(v & 0xFFFFu)), dense_to_f32<TYPE>((uint16_t)(v >> 16)));
}

// 1 / (1 + exp(-v)) by the hardware's exp2 and reciprocal (relative error about 1e-6, a bf16 half step is 4e-3, an fp16 one
// 5e-4); 1 at +inf, 0 at -inf and from -87.4 down, where it is below fp32's normal numbers; NaN stays.
__device__ __forceinline__ float dense_sigmoid(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}

// tanh: beyond 1/4 through the same two instructions, 1 - 2 / (1 + exp(2 y)); below, where that would lose digits, by its
// Taylor series to y^9 (the first term left out is 9e-9 of the value at 1/4).
__device__ __forceinline__ float dense_tanh(float y) {
  const float q = y * y;
  const float near = y * (1.0f + q * (-0.33333333f + q * (0.13333333f + q * (-0.053968254f + q * 0.021869489f))));
  const float far = 1.0f - 2.0f * dense_sigmoid(-2.0f * y);
  return fabsf(y) < 0.25f ? near : far;
}
// The normal distribution up to z and e = exp(-z^2 / 2): erfc(x) exp(x^2) = t (a1 + a2 t + .. + a7 t^6), t = 1 / (1 + 0.375 x),
// x = |z| / sqrt(2) - the form of Abramowitz and Stegun 7.1.26, which keeps erfc's absolute error small; these coefficients are
// fitted to its relative error (Remez's exchange, 0 <= x <= 9.8: 6.4e-7), so that the tail is good to its last digits too. On top
// comes the rounding of e's argument, z^2 2^-23 of the value: 8e-6 at -13, where bf16 ends.
__device__ __forceinline__ float dense_normal_cdf(float z, float& e) {
  float t;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * z * -0.72134752f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.375f * 0.70710678f, fabsf(z), 1.0f)));
  const float q = 0.5f * e * t * (0.21133944f + t * (0.21568918f + t * (0.16666456f + t * (0.28306156f + t * (-0.12959732f + t * (0.3879378f + t * -0.13509591f))))));
  return z < 0.0f ? q : 1.0f - q;
}

constexpr float kInvSqrt2Pi = 0.39894228040143268f;
// 0.5 (1 + tanh(y)) = sigmoid(2 y), y = sqrt(2 / pi) (z + 0.044715 z^3)
constexpr float kGeluC = 1.5957691216057308f, kGeluA = 0.044715f;

// Activation of the linear projection.
__device__ __forceinline__ float dense_act(int act, float z) {
  switch (act) {
    case kActSilu: return z * dense_sigmoid(z);
    case kActGelu: {
      float e;
      return z * dense_normal_cdf(z, e);
    }
    case kActGeluTanh: return z * dense_sigmoid(kGeluC * (z + kGeluA * z * z * z));
    default: return z;
  }
}
// Its slope, finite for every finite z: z z is kept below 1e8 where it stands beside 1 - p, which is 0 long before.
__device__ __forceinline__ float dense_act_slope(int act, float z) {
  switch (act) {
    case kActSilu: {
      const float p = dense_sigmoid(z);
      return p + z * p * (1.0f - p);
    }
    case kActGelu: {
      float e;
      const float cdf = dense_normal_cdf(z, e);
      return cdf + z * kInvSqrt2Pi * e;
    }
    case kActGeluTanh: {
      const float p = dense_sigmoid(kGeluC * (z + kGeluA * z * z * z));
      return p + z * p * (1.0f - p) * kGeluC * (1.0f + 3.0f * kGeluA * fminf(z * z, 1e8f));
    }
    default: return 1.0f;
  }
}

// tanh(y) as a quotient n / (e + 1), e = exp(2 y) = 2^t: n = e - 1, or below 1/32, where that would lose digits,
// (e + 1) (y - y^3 / 3) (the next term is 1e-7 of the value). t is kept below 29, where tanh is 1 to the last bit.
__device__ __forceinline__ float dense_tanh_parts(float t, float& e) {
  constexpr float kHalfLn2 = 0.34657359f;      // y = t ln(2) / 2
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(t) : "f"(29.0f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  const float near = t * fmaf(t * t, -kHalfLn2 * kHalfLn2 * kHalfLn2 / 3.0f, kHalfLn2) * (e + 1.0f);
  return fabsf(t) < 0.09f ? near : e - 1.0f;
}

// The gated product of one feature. min.NaN / max.NaN: a NaN stays NaN. SiTU's three quotients - two tanh, one sigmoid - have one
// reciprocal: three exp2 and it are what the special-function unit does for an element (333 x 2880 -> 2880: a reciprocal and a
// division for each took 2.5 us longer). The denominators' product passes fp32's range - 2^29 from up's tanh alone, exp(-g) from
// the sigmoid - so the sigmoid's is taken 2^-60 times, and k.scale holds the 2^-60 that takes it back: the quotient becomes 0 only
// where exp(-g) times up's denominator passes 2^186, from g = -109 on for the largest up, where the sigmoid is 5e-48.
__device__ __forceinline__ float dense_gated(int act, float g, float u, const GatedKind& k) {
  if (act == 1) {
    float e1, e2, e3 = 0.0f, r, n3 = k.scale, last = u;
    const float n1 = dense_tanh_parts(g * k.t_beta, e1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e2) : "f"(fmaf(g, -1.4426950408889634f, -(float)kSituLift)));
    if (k.linear_beta > 0.0f) {
      n3 = dense_tanh_parts(u * k.t_linear, e3);
      last = k.scale;
    }
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((e1 + 1.0f) * (e2 + kSituLifted) * (e3 + 1.0f)));
    return n1 * r * n3 * last;
  }
  const float limit = k.limit, lo = -limit;
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(g) : "f"(limit));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(u) : "f"(limit));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(u) : "f"(lo));
  return g * dense_sigmoid(g) * u;
}
// Its gradient with respect to both pre-activations, for the gradient dh of the product.
__device__ __forceinline__ void dense_gated_grad(int act, float dh, float g, float u, const GatedKind& k, float& dg, float& du) {
  if (act == 1) {
    const bool bent = k.linear_beta > 0.0f;
    const float p = dense_sigmoid(g), a = dense_tanh(g * k.inv_beta), b = bent ? dense_tanh(u * k.inv_linear_beta) : 0.0f;
    const float up = bent ? k.linear_beta * b : u;
    dg = dh * up * ((1.0f - a * a) * p + k.beta * a * p * (1.0f - p));
    du = dh * (k.beta * a * p) * (1.0f - b * b);
    return;
  }
  const float limit = k.limit, lo = -limit;
  float gc = g, uc = u;
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(gc) : "f"(limit));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(uc) : "f"(limit));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(uc) : "f"(lo));
  const float p = dense_sigmoid(gc), gate = gc * p;
  dg = g > limit ? 0.0f : dh * uc * (p + gate * (1.0f - p));
  du = fabsf(u) > limit ? 0.0f : dh * gate;
}

// Column sums of the chunks by eight warps as the `cta`-th of `ctas`: 32 columns at a time, each warp an eighth of the chunks, 16
// loads on their way; the eighths in order.
template <int TYPE>
__device__ __forceinline__ void sum_chunks(const DenseSums& q, int cta, int ctas, int warp, int lane, float (*room)[32]) {
  const int first = (int)((int64_t)q.chunks * warp / 8), end = (int)((int64_t)q.chunks * (warp + 1) / 8);
#pragma unroll 1
  for (int c = cta * 32 + lane; c - lane < q.cols; c += ctas * 32) {
    float s = 0.0f;
#pragma unroll 1
    for (int i = first; i < end; i += 16) {
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = i + j < end && c < q.cols ? q.partial[(int64_t)(i + j) * q.cols + c] : 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) s += v[j];
    }
    room[warp][lane] = s;
    __syncwarp();   // bar.sync takes a warp's lanes as one; those behind the last column have not loaded
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (warp == 0 && c < q.cols) {
      s = room[0][lane];
#pragma unroll
      for (int i = 1; i < 8; ++i) s += room[i][lane];
      q.db[c] = dense_from_f32<TYPE>(s);
    }
    __syncwarp();
    asm volatile("bar.sync 1, 256;" ::: "memory");
  }
}

}  // namespace

}  // namespace vkernels::kernels::cuda
