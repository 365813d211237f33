// What the kernels over rows of logits share: element types, the temperature, the order of values.
#pragma once
#include "ctx.h"
#include "ptx.cuh"
#include "vocab_rows.h"

namespace rt {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// max that lets a NaN through
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// d / T for d = z - max <= 0, correctly rounded but for the last bit: the reciprocal alone would be off by half a step of d / T,
// the same way for every element.  Below -200 T the exponential is 0 whatever d is, -inf among them, which the
// correction would turn into NaN.
struct Temperature {
  float t, inv;
  __device__ __forceinline__ explicit Temperature(float t_) : t(t_), inv(1.0f / t_) {}
  __device__ __forceinline__ float operator()(float d) const {
    d = fmaxf(d, -200.0f * t);
    const float x = d * inv;
    return t == 1.0f ? d : fmaf(fmaf(-x, t, d), inv, x);
  }
};

// Integers in the order of the values: NaN above all, the two zeros alike.
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 becomes +0
  if (v != v) return 0xffffffffu;
  return b ^ (uint32_t)(((int32_t)b >> 31) | 0x80000000);
}
__device__ __forceinline__ float order32_value(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);  // the highest one, a NaN's, is a NaN
}

// Calls f with a null pointer of the element type that `dtype` names.
template <class F>
inline int with_dtype(int dtype, F&& f) {
  if (dtype == RT_DT_F32) return f((float*)nullptr);
  if (dtype == RT_DT_BF16) return f((__nv_bfloat16*)nullptr);
  return f((__half*)nullptr);
}

}  // namespace rt
