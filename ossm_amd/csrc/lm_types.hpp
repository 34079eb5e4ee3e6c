// Element types, activations and small helpers shared by the language-model operators.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ossm {
namespace {

struct bf16_t {
  uint16_t bits;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16_t v) { return __uint_as_float(static_cast<uint32_t>(v.bits) << 16); }

template <class E>
__device__ __forceinline__ E from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16_t from_f<bf16_t>(float v) {  // to nearest, ties to even
  const __bf16 b = static_cast<__bf16>(v);
  return bf16_t{__builtin_bit_cast(uint16_t, b)};
}

// The hardware reciprocal (within 1 ulp): the exact division's ten instructions were a sixth
// of the scans' time outside their states.
__device__ __forceinline__ float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }
__device__ __forceinline__ float silu_f(float x) { return x * sigmoid_f(x); }

// softplus(x) = max(x, 0) + log1p(exp(-|x|)), the logarithm by its series in
// z = e / (2 + e) <= 1/3, log1p(e) = 2 (z + z^3/3 + ...): the terms left out are below
// 2^-25 of the sum, and tiny e keep their relative accuracy (the hardware logarithm of
// 1 + e would not).
__device__ __forceinline__ float softplus_f(float x) {
  const float e = __expf(-fabsf(x));
  const float z = e * __builtin_amdgcn_rcpf(2.f + e), q = z * z;
  float s = 1.f / 15.f;
  s = fmaf(s, q, 1.f / 13.f);
  s = fmaf(s, q, 1.f / 11.f);
  s = fmaf(s, q, 1.f / 9.f);
  s = fmaf(s, q, 1.f / 7.f);
  s = fmaf(s, q, 1.f / 5.f);
  s = fmaf(s, q, 1.f / 3.f);
  s = fmaf(s, q, 1.f);
  return fmaxf(x, 0.f) + 2.f * z * s;
}

}  // namespace
}  // namespace ossm
