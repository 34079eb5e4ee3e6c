// Vectors of a row at any address, and sums over groups of lanes, shared by the
// language-model operators whose rows start anywhere.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "lm_types.hpp"

namespace ossm {
namespace {

// W elements that need no more than the element's own alignment: gfx950 reads and writes
// such a vector in one instruction at any address, so that rows of odd sizes (each starting at another
// offset) keep wide accesses.
template <class E, int W>
struct __attribute__((packed, aligned(alignof(E)))) Loose {
  E v[W];
};

template <class E, int W>
__device__ __forceinline__ void load_loose(const E* p, E (&v)[W]) {
  const Loose<E, W> t = *reinterpret_cast<const Loose<E, W>*>(p);
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] = t.v[k];
}

template <class E, int W>
__device__ __forceinline__ void store_loose(E* p, const E (&v)[W]) {
  Loose<E, W> t;
#pragma unroll
  for (int k = 0; k < W; ++k) t.v[k] = v[k];
  *reinterpret_cast<Loose<E, W>*>(p) = t;
}

// The first n (0 .. W) elements at p, zeros behind them.
template <class E, int W>
__device__ __forceinline__ void load_part(const E* p, int n, E (&v)[W]) {
  if (n >= W) {
    load_loose(p, v);
    return;
  }
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] = k < n ? p[k] : from_f<E>(0.f);
}

template <class E, int W>
__device__ __forceinline__ void store_part(E* p, int n, const E (&v)[W]) {
  if (n >= W) {
    store_loose(p, v);
    return;
  }
#pragma unroll
  for (int k = 0; k < W; ++k)
    if (k < n) p[k] = v[k];
}

// Sum over the G lanes (a power of two up to 64) of the calling lane's group, the same in
// each and in a fixed order.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

}  // namespace
}  // namespace ossm
