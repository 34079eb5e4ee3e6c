// Vectors of a row at any address, and sums over groups of lanes, shared by the
// language-model operators whose rows start anywhere.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "lm_types.hpp"

namespace ossm {
namespace {

// W elements in whole registers, two 16-bit ones each (as an array of its elements a vector
// in flight would hold every one in a register of its own).
template <class E, int W>
struct Vec {
  static constexpr int kWords = W * static_cast<int>(sizeof(E)) / 4;
  // needs no more than the element's own alignment: gfx950 reads and writes it in one instruction
  // at any address, so that rows of odd sizes keep wide accesses
  typedef uint32_t Loose __attribute__((ext_vector_type(kWords), aligned(alignof(E))));
  uint32_t w[kWords];

  __device__ __forceinline__ float get(int k) const {
    if constexpr (sizeof(E) == 4) return __uint_as_float(w[k]);
    else return __uint_as_float(k % 2 == 0 ? w[k / 2] << 16 : w[k / 2] & 0xffff0000u);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void set(const float (&v)[W]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(E) == 4) w[i] = __float_as_uint(v[i]);
      else w[i] = static_cast<uint32_t>(from_f<bf16_t>(v[2 * i]).bits) | static_cast<uint32_t>(from_f<bf16_t>(v[2 * i + 1]).bits) << 16;
    }
  }
  // the first n (1 and on) elements at p, of which `room` may be read; what lies behind the
  // n is left to keep(), so that nothing waits for the load
  __device__ __forceinline__ void load(const E* p, int n, long long room = 0) {
    if (n >= W || room >= W) {
      const Loose t = *reinterpret_cast<const Loose*>(p);
      __builtin_memcpy(w, &t, sizeof(t));
      return;
    }
    float v[W];
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = k < n ? to_f(p[k]) : 0.f;
    set(v);
  }
  __device__ __forceinline__ void keep(int n) {  // zeros behind the first n
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(E) == 4) w[i] = i < n ? w[i] : 0u;
      else w[i] &= 2 * i + 1 < n ? 0xffffffffu : 2 * i < n ? 0xffffu : 0u;
    }
  }
  // the first n to p; kOnce past the caches, for what is written once and read by later
  // kernels only (not where rows share lines: each would be written twice).  A choice between
  // the two at run time would be one plain store to the compiler.
  template <bool kOnce>
  __device__ __forceinline__ void store(E* p, int n) const {
    if (n >= W) {
      Loose t;
      __builtin_memcpy(&t, w, sizeof(t));
      if constexpr (kOnce) __builtin_nontemporal_store(t, reinterpret_cast<Loose*>(p));
      else *reinterpret_cast<Loose*>(p) = t;
      return;
    }
    part(p, n);
  }

 private:
  __device__ __forceinline__ void part(E* p, int n) const {
#pragma unroll
    for (int k = 0; k < W; ++k)
      if (k < n) p[k] = from_f<E>(get(k));  // exact: the value is one of E's
  }
};

// Sum over the G lanes (a power of two up to 64) of the calling lane's group, the same in
// each and in a fixed order.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Sum of column i of `partial` [n, ld], by a workgroup of 1024 threads for its 16 columns
// (blockIdx.x 16 and on): 64 threads a column, each every 64th row, four of them in
// flight, in 64 bits and in a fixed order.  Few columns of many rows would leave most CUs
// without work at 64 columns a workgroup ([1024, 2048]: 29 us against 9).  Threads 0 to 15 get their column's.
constexpr int kSumThreads = 1024, kSumColumns = 16;
__device__ __forceinline__ double column_sum(const float* partial, int n, long long ld, long long cols) {
  constexpr int kEach = kSumThreads / kSumColumns;
  __shared__ double s_sum[kEach][kSumColumns];
  const int c = threadIdx.x % kSumColumns, r0 = threadIdx.x / kSumColumns;
  const long long i = static_cast<long long>(blockIdx.x) * kSumColumns + c;
  double t[4] = {};
  if (i < cols) {
    int r = r0;
    for (; r + 3 * kEach < n; r += 4 * kEach) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = partial[(r + static_cast<long long>(k) * kEach) * ld + i];
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] += v[k];
    }
    for (; r < n; r += kEach) t[0] += partial[r * ld + i];
  }
  s_sum[r0][c] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
#pragma unroll
  for (int o = kEach / 2; o > 0; o >>= 1) {
    if (r0 < o) s_sum[r0][c] += s_sum[r0 + o][c];
    __syncthreads();
  }
  return s_sum[0][c];
}

}  // namespace
}  // namespace ossm
