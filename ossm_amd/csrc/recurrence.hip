// The gated linear recurrence, forward and backward over batches of sequences, over
// packed ragged prompts with states in a pool, and over single tokens
// (ossm_recurrence_forward, _backward, _prompt, _step).  Per channel d:
//
//   l_t = -scale softplus(decay_d) sigmoid(r_t),  a_t = exp(l_t)
//   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t,   y_t = h_t, or h_t silu(z_t)
//
// The input's factor is sqrt(-expm1(2 l)): 1 - a^2 of a rounded a near one would keep few
// digits of it.  The backward, G_t the gradient that reaches h_t:
//
//   G_t = gy_t silu(z_t) + a_{t+1} G_{t+1},   gz = gy h silu'(z)
//   gx = G m g,  gi = G m x g (1 - g),   m = sqrt(1 - a^2), g = sigmoid(i)
//   q = l dL/dl = G (a l h_{t-1} + g x a^2 (-l) / m),   gr = q (1 - sigmoid(r))
//   gdecay = sigmoid(decay) / softplus(decay) sum of q
//
// It is bound by memory (a few bytes and some fifty operations an element), so each tensor is
// read once: time is cut into chunks of T W steps, a workgroup of W waves takes a chunk of
// 64 V channels (V a lane), wave w its steps from w T on.  Each wave folds its steps into
// one (sum of l, state from zero), the waves are joined through LDS, and the chunk's start comes
// from the chunks before it by records in the stream's scratch.  A chunk's place among W
// neighbours is fixed: it waits for the aggregates of its neighbours before it, a
// wave each, and for the state at the end of the W before them, so the wait is one round
// trip for W chunks, and every sum has one order: results are bitwise repeatable.
//
// Decays over several steps are kept as sums of l and applied in two halves: exp(l) of a
// chunk underflows where its product with a state need not, and neither half goes below the smallest
// normal number, so that an infinite state stays infinite.

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <string>

#include "../../include/ossm_lm.h"
#include "lm_types.hpp"
#include "lm_vector.hpp"
#include "runtime.hpp"
#include "scan_device.hpp"

namespace ossm {
namespace {

constexpr int kSteps = 8, kWaves = 16, kBackWaves = 8;  // chunks of 128 steps, in the backward of 64
constexpr int kSavedEvery = kSteps * kBackWaves;

constexpr float kTiny = 1.17549435e-38f;  // the smallest normal number

// ---- the step's values ----------------------------------------------------------
// exp(x) for x <= 0 or moderate: the rounding of x log2(e) is put back, so that the
// result is good to 2^-22 at any x (the bare instruction loses |x| 2^-24).
__device__ __forceinline__ float exp_f(float x) {
  const float y = x * 1.44269504f;
  const float rest = fmaf(x, 1.44269504f, -y) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(y);
  return fmaf(e, rest * 0.693147181f, e);
}

// NaN passes through the least and the greatest of two, which fminf and fmaxf would drop.
__device__ __forceinline__ float least(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float greatest(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The reciprocal is the hardware's, within 1 ulp.  Bounds keep infinities out of exp_f.
__device__ __forceinline__ float sigmoid_exact(float x) {
  return __builtin_amdgcn_rcpf(1.f + exp_f(greatest(least(-x, 88.f), -88.f)));
}

// a and m = sqrt(1 - a^2) of a log-decay l <= 0.  Near zero 1 - a^2 = -expm1(2 l) by its
// series (left out: below 2^-24 of it), from -0.2 on a^2 is far enough from one.
__device__ __forceinline__ void decay_of(float l, float& a, float& m) {
  a = greatest(exp_f(greatest(l, -200.f)), kTiny);
  const float q = l + l;
  float s = 1.f / 5040.f;
  s = fmaf(s, q, 1.f / 720.f);
  s = fmaf(s, q, 1.f / 120.f);
  s = fmaf(s, q, 1.f / 24.f);
  s = fmaf(s, q, 1.f / 6.f);
  s = fmaf(s, q, 0.5f);
  s = fmaf(s, q, 1.f);
  m = __builtin_amdgcn_sqrtf(q > -0.4f ? -q * s : fmaf(-a, a, 1.f));
}

// exp(l) h, in two halves.  -inf means that nothing before counts, whatever it holds.
__device__ __forceinline__ float decayed(float l, float h) {
  const float e = greatest(exp_f(greatest(0.5f * l, -200.f)), kTiny);
  return l == -__builtin_inff() ? 0.f : (h * e) * e;
}

// scale softplus(decay), and sigmoid(decay) / softplus(decay)
__device__ __forceinline__ float decay_rate(float decay, float scale) {
  return scale * (fmaxf(decay, 0.f) + log1pf(expf(-fabsf(decay))));
}

__global__ void decay_grad_kernel(const float* partial, int n, int D, const float* decay, float* out) {
  __shared__ double s_sum[16][64];
  const int i = static_cast<int>(blockIdx.x) * 64 + threadIdx.x % 64, w = threadIdx.x / 64;
  double t = 0;
  if (i < D)
    for (int r = w; r < n; r += 16) t += partial[static_cast<size_t>(r) * D + i];
  s_sum[w][threadIdx.x % 64] = t;
  __syncthreads();
  if (w != 0 || i >= D) return;
  for (int v = 1; v < 16; ++v) t += s_sum[v][threadIdx.x];
  const double x = decay[i];
  // sigmoid / softplus goes to one below; past -40 the quotient's own terms vanish
  const double ratio = x < -40 ? 1. : 1. / ((1. + exp(-x)) * (fmax(x, 0.) + log1p(exp(-fabs(x)))));
  out[i] = static_cast<float>(t * ratio);
}

// ---- records ------------------------------------------------------------------------
// Per chunk and channel: the aggregate's sum of l and state, and the state at the
// chunk's end (written by the last chunk of W neighbours only).
enum { kSumL = 0, kState = 1, kEnd = 2, kRecords = 3 };

struct Rec {
  unsigned long long* base;
  size_t channels;
  __device__ __forceinline__ unsigned long long* at(int chunk, int word, size_t ch) const {
    return base + (static_cast<size_t>(chunk) * kRecords + word) * channels + ch;
  }
};

template <int V>
__device__ __forceinline__ void publish(unsigned long long* p, const float (&v)[V], unsigned tag) {
#pragma unroll
  for (int k = 0; k < V; ++k)
    __hip_atomic_store(p + k, static_cast<unsigned long long>(tag) << 32 | __float_as_uint(v[k]), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

// Waits for V tagged words each at p and q (q may be null); NaN where the wait gives up.
template <int V>
__device__ __forceinline__ void await(const unsigned long long* p, const unsigned long long* q, const LaunchSync& sync,
                                      float (&vp)[V], float (&vq)[V]) {
  const float nan = __builtin_nanf("");
#pragma unroll
  for (int k = 0; k < V; ++k) vp[k] = vq[k] = nan;
  if (sync.poison) return;
  for (uint32_t spins = 0;; ++spins) {
    unsigned long long a[V], b[V];
    bool ok = true;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      a[k] = __hip_atomic_load(p + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      b[k] = q != nullptr ? __hip_atomic_load(q + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : a[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k)
      ok = ok && static_cast<unsigned>(a[k] >> 32) == sync.tag && static_cast<unsigned>(b[k] >> 32) == sync.tag;
    if (ok) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        vp[k] = __uint_as_float(static_cast<unsigned>(a[k]));
        vq[k] = __uint_as_float(static_cast<unsigned>(b[k]));
      }
      return;
    }
    if (spins > kSpinLimit) {
      __hip_atomic_fetch_or(sync.err, kErrSpinTimeout, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return;
    }
    __builtin_amdgcn_s_sleep(2);
  }
}

// One workgroup's part of the scan between chunks.  j: the chunk's place in time order
// of the scan (for the backward counted from the end), l and h the calling wave's
// aggregate; start: the state before the first chunk.  Returns the state from which the
// calling wave starts; waves are in scan order.
template <int V, int W>
struct Join {
  float l[W][64][V], h[W][64][V];    // the waves' aggregates
  float pl[W][64][V], ph[W][64][V];  // what the chunks before hand over
};

template <int V, int W>
__device__ __forceinline__ void join_chunks(Join<V, W>& s, int w, int lane, int j, int n_chunks, const Rec& rec, size_t ch,
                                            const LaunchSync& sync, float (&l)[V], float (&h)[V], const float (&start)[V],
                                            float (&carry)[V]) {
  const int place = j % W;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    s.l[w][lane][k] = l[k];
    s.h[w][lane][k] = h[k];
  }
  __syncthreads();
  const bool more = j + 1 < n_chunks;
  if (more && place + 1 < W && w == W - 1) {  // the chunk's aggregate, for its neighbours
    float al[V], ah[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      al[k] = s.l[0][lane][k];
      ah[k] = s.h[0][lane][k];
#pragma unroll
      for (int v = 1; v < W; ++v) {
        const float d = s.l[v][lane][k];
        ah[k] = decayed(d, ah[k]) + s.h[v][lane][k];
        al[k] = d == -__builtin_inff() ? d : al[k] + d;
      }
    }
    publish<V>(rec.at(j, kSumL, ch), al, sync.tag);
    publish<V>(rec.at(j, kState, ch), ah, sync.tag);
  }
  if (j > 0) {
    float a[V] = {}, b[V] = {};
    if (w < place) await<V>(rec.at(j - place + w, kSumL, ch), rec.at(j - place + w, kState, ch), sync, a, b);
    else if (w == place && j > place) await<V>(rec.at(j - place - 1, kEnd, ch), nullptr, sync, a, b);
    if (w <= place) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        s.pl[w][lane][k] = a[k];
        s.ph[w][lane][k] = b[k];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    float c = j > place ? s.ph[place][lane][k] : start[k];
    for (int v = 0; v < place; ++v) c = decayed(s.pl[v][lane][k], c) + s.ph[v][lane][k];
    for (int v = 0; v < w; ++v) c = decayed(s.l[v][lane][k], c) + s.h[v][lane][k];
    carry[k] = c;
  }
  if (more && place == W - 1 && w == W - 1) {
    float end[V];
#pragma unroll
    for (int k = 0; k < V; ++k) end[k] = decayed(l[k], carry[k]) + h[k];
    publish<V>(rec.at(j, kEnd, ch), end, sync.tag);
  }
}

// ---- forward ----------------------------------------------------------------------------
template <class E>
struct Forward {
  const E* x;
  const E* i;
  const E* r;
  const E* z;
  long long ld_x, ld_i, ld_r, ld_z;
  const float* decay;
  float scale;
  const float* start;  // [B, D] or null
  E* y;
  float* last;   // [B, D]
  float* saved;  // [B, n_saved, D] the state before each of the backward's chunks, or null
  // packed prompts
  float* pool;
  const int32_t* slots;
  const int32_t* out_slots;
  const int32_t* offsets;
  const uint8_t* resume;
  int n_seqs, n_slots;
  int B, L, D, n_cols, n_chunks, n_saved;
};

template <class E, int V>
struct alignas(V * sizeof(E)) Lane {
  E v[V];
};

template <class E, int V>
__device__ __forceinline__ Lane<E, V> lane_load(const E* p) {
  return *reinterpret_cast<const Lane<E, V>*>(p);
}

// h of a prompt before its first token
template <class E, int V>
__device__ __forceinline__ void prompt_start(const Forward<E>& g, int seq, int ch, float (&h)[V]) {
  const int slot = g.resume != nullptr && g.resume[seq] ? g.slots[seq] : -1;
#pragma unroll
  for (int k = 0; k < V; ++k)
    h[k] = slot >= 0 && slot < g.n_slots ? g.pool[static_cast<size_t>(slot) * g.D + ch + k] : 0.f;
}

template <class E, int V>
__device__ __forceinline__ void prompt_end(const Forward<E>& g, int seq, int ch, bool active, const float (&h)[V]) {
  const int slot = g.out_slots[seq];
  if (!active || slot < 0 || slot >= g.n_slots) return;
#pragma unroll
  for (int k = 0; k < V; ++k) g.pool[static_cast<size_t>(slot) * g.D + ch + k] = h[k];
}

template <class E, int V, int T, int W, bool PACKED>
__global__ __launch_bounds__(W * 64) void recurrence_forward_kernel(Forward<E> g, unsigned long long* records, LaunchSync sync) {
  __shared__ Join<V, W> s_join;
  __shared__ int s_first[PACKED ? T * W : 1], s_final[PACKED ? T * W : 1];  // the prompt that starts, ends at a token, + 1
  __shared__ int s_ticket;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int n_groups = g.B * g.n_cols;
  const int ticket = launch_order(sync, n_groups * g.n_chunks, &s_ticket);
  const int c = ticket / n_groups, group = ticket - c * n_groups;
  const int seq = group / g.n_cols, col = group - seq * g.n_cols;
  const int ch_raw = (col * 64 + lane) * V;
  const bool active = ch_raw < g.D;
  const int ch = active ? ch_raw : g.D - V;  // past the end: the last channels, never stored
  const int t_chunk = c * T * W, t0 = t_chunk + w * T;
  const long long row0 = static_cast<long long>(seq) * g.L;

  Lane<E, V> x[T], in[T], r[T], z[T];
#pragma unroll
  for (int k = 0; k < T; ++k) {
    const long long row = row0 + min(t0 + k, max(g.L - 1, 0));
    if (g.L > 0) {
      r[k] = lane_load<E, V>(g.r + row * g.ld_r + ch);
      in[k] = lane_load<E, V>(g.i + row * g.ld_i + ch);
      x[k] = lane_load<E, V>(g.x + row * g.ld_x + ch);
      if (g.z != nullptr) z[k] = lane_load<E, V>(g.z + row * g.ld_z + ch);
    }
  }
  if constexpr (PACKED) {
    for (int k = threadIdx.x; k < T * W; k += W * 64) s_first[k] = s_final[k] = 0;
    __syncthreads();
    // a stretch of prompts a thread: only one whose tokens meet the chunk's is looked through
    const int span = (g.n_seqs + W * 64 - 1) / (W * 64), lo = min(static_cast<int>(threadIdx.x) * span, g.n_seqs);
    const int hi = min(lo + span, g.n_seqs);
    if (lo < hi && g.offsets[lo] < t_chunk + T * W && g.offsets[hi] >= t_chunk) {
      for (int s = lo; s < hi; ++s) {
        const int a = g.offsets[s], b = g.offsets[s + 1];
        if (a >= b) continue;
        if (a >= t_chunk && a < t_chunk + T * W) s_first[a - t_chunk] = s + 1;
        if (b - 1 >= t_chunk && b - 1 < t_chunk + T * W) s_final[b - 1 - t_chunk] = s + 1;
      }
    }
    // empty prompts hand on the state that they start from, a share of them a chunk
    for (int s = c * W + w; s < g.n_seqs; s += g.n_chunks * W) {
      if (g.offsets[s] < g.offsets[s + 1]) continue;
      float h[V];
      prompt_start<E, V>(g, s, ch, h);
      prompt_end<E, V>(g, s, ch, active, h);
    }
    __syncthreads();
  }
  float rate[V], a[T][V], b[T][V], sum[V], h[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    rate[k] = -decay_rate(g.decay[ch + k], g.scale);
    sum[k] = h[k] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < T; ++k) {
    const int first = PACKED ? __builtin_amdgcn_readfirstlane(s_first[w * T + k]) : 0;
    float init[V];
    if (PACKED && first != 0) prompt_start<E, V>(g, first - 1, ch, init);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float l = rate[v] * sigmoid_exact(to_f(r[k].v[v])), m;
      decay_of(l, a[k][v], m);
      b[k][v] = m * sigmoid_exact(to_f(in[k].v[v])) * to_f(x[k].v[v]);
      if (t0 + k >= g.L) {  // past the end: nothing changes
        a[k][v] = 1.f;
        b[k][v] = l = 0.f;
      }
      if (PACKED && first != 0) {
        b[k][v] = fmaf(a[k][v], init[v], b[k][v]);
        a[k][v] = -1.f;  // nothing before counts
        sum[v] = -__builtin_inff();
        h[v] = b[k][v];
      } else {
        sum[v] = sum[v] == -__builtin_inff() ? sum[v] : sum[v] + l;
        h[v] = fmaf(a[k][v], h[v], b[k][v]);
      }
    }
  }
  const Rec rec{records, static_cast<size_t>(n_groups) * 64 * V};
  const size_t rec_ch = (static_cast<size_t>(group) * 64 + lane) * V;
  float start[V], carry[V];
#pragma unroll
  for (int k = 0; k < V; ++k) start[k] = !PACKED && g.start != nullptr ? g.start[static_cast<size_t>(seq) * g.D + ch + k] : 0.f;
  join_chunks<V, W>(s_join, w, lane, c, g.n_chunks, rec, rec_ch, sync, sum, h, start, carry);

  if (!PACKED && g.saved != nullptr && t0 % kSavedEvery == 0 && t0 < g.L && active) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      g.saved[(static_cast<size_t>(seq) * g.n_saved + t0 / kSavedEvery) * g.D + ch + k] = carry[k];
  }
  const int lo = PACKED ? (g.n_seqs > 0 ? g.offsets[0] : 0) : 0, hi = PACKED ? (g.n_seqs > 0 ? g.offsets[g.n_seqs] : 0) : 0;
#pragma unroll
  for (int k = 0; k < T; ++k) {
    if (t0 + k >= g.L) break;
    Lane<E, V> out;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      carry[v] = PACKED && a[k][v] < 0.f ? b[k][v] : fmaf(a[k][v], carry[v], b[k][v]);
      float y = carry[v];
      if (g.z != nullptr) {
        const float zz = to_f(z[k].v[v]);
        y *= zz * sigmoid_exact(zz);
      }
      if (PACKED && (t0 + k < lo || t0 + k >= hi)) y = 0.f;
      out.v[v] = from_f<E>(y);
    }
    if (active) *reinterpret_cast<Lane<E, V>*>(g.y + (row0 + t0 + k) * g.D + ch) = out;
    if constexpr (PACKED) {
      const int final = __builtin_amdgcn_readfirstlane(s_final[w * T + k]);
      if (final != 0) prompt_end<E, V>(g, final - 1, ch, active, carry);
    } else if (t0 + k == g.L - 1 && active) {
#pragma unroll
      for (int v = 0; v < V; ++v) g.last[static_cast<size_t>(seq) * g.D + ch + v] = carry[v];
    }
  }
}

// ---- backward ---------------------------------------------------------------------------
template <class E>
struct Backward {
  const E* x;
  const E* i;
  const E* r;
  const E* z;
  const E* gy;
  long long ld_x, ld_i, ld_r, ld_z, ld_gy, ld_out;
  const float* decay;
  float scale;
  const float* saved;  // [B, n_chunks, D]
  const float* glast;  // [B, D] or null
  E* gx;
  E* gi;
  E* gr;
  E* gz;
  float* gstart;   // [B, D] or null
  float* partial;  // [n_chunks B, D] sums of q
  int B, L, D, n_cols, n_chunks;
};

template <class E, int V, int T, int W>
__global__ __launch_bounds__(W * 64) void recurrence_backward_kernel(Backward<E> g, unsigned long long* records, LaunchSync sync) {
  __shared__ Join<V, W> s_join;
  __shared__ float s_l[W][64][V], s_h[W][64][V];
  __shared__ int s_ticket;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int n_groups = g.B * g.n_cols;
  const int ticket = launch_order(sync, n_groups * g.n_chunks, &s_ticket);
  const int j = ticket / n_groups, group = ticket - j * n_groups;
  const int c = g.n_chunks - 1 - j;  // the last chunk first
  const int seq = group / g.n_cols, col = group - seq * g.n_cols;
  const int ch_raw = (col * 64 + lane) * V;
  const bool active = ch_raw < g.D;
  const int ch = active ? ch_raw : g.D - V;
  const int t0 = c * T * W + w * T;
  const long long row0 = static_cast<long long>(seq) * g.L;

  Lane<E, V> x[T], in[T], r[T], z[T], gy[T];
#pragma unroll
  for (int k = 0; k < T; ++k) {
    const long long row = row0 + min(t0 + k, g.L - 1);
    r[k] = lane_load<E, V>(g.r + row * g.ld_r + ch);
    in[k] = lane_load<E, V>(g.i + row * g.ld_i + ch);
    x[k] = lane_load<E, V>(g.x + row * g.ld_x + ch);
    gy[k] = lane_load<E, V>(g.gy + row * g.ld_gy + ch);
    if (g.z != nullptr) z[k] = lane_load<E, V>(g.z + row * g.ld_z + ch);
  }
  float rate[V], a[T][V], b[T][V], sum[V], h[V], M[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = -decay_rate(g.decay[ch + v], g.scale);
    sum[v] = h[v] = M[v] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < T; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float l = rate[v] * sigmoid_exact(to_f(r[k].v[v])), m;
      decay_of(l, a[k][v], m);
      b[k][v] = m * sigmoid_exact(to_f(in[k].v[v])) * to_f(x[k].v[v]);
      if (t0 + k >= g.L) {
        a[k][v] = 1.f;
        b[k][v] = l = 0.f;
      }
      sum[v] += l;
      h[v] = fmaf(a[k][v], h[v], b[k][v]);
    }
  const auto upstream = [&](int k, int v) {
    float o = t0 + k < g.L ? to_f(gy[k].v[v]) : 0.f;
    if (g.z != nullptr) {
      const float zz = to_f(z[k].v[v]);
      o *= zz * sigmoid_exact(zz);
    }
    return o;
  };
  // what reaches the step before the wave's first, from a zero gradient behind its last
#pragma unroll
  for (int k = T - 1; k >= 0; --k)
#pragma unroll
    for (int v = 0; v < V; ++v) M[v] = a[k][v] * (upstream(k, v) + M[v]);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s_l[w][lane][v] = sum[v];
    s_h[w][lane][v] = h[v];
  }
  const Rec rec{records, static_cast<size_t>(n_groups) * 64 * V};
  const size_t rec_ch = (static_cast<size_t>(group) * 64 + lane) * V;
  float start[V], carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) start[v] = g.glast != nullptr ? g.glast[static_cast<size_t>(seq) * g.D + ch + v] : 0.f;
  // the waves in the scan's order: the last first
  join_chunks<V, W>(s_join, W - 1 - w, lane, j, g.n_chunks, rec, rec_ch, sync, sum, M, start, carry);

  // the states again, from the chunk's start
  float before[T][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float s = g.saved[(static_cast<size_t>(seq) * g.n_chunks + c) * g.D + ch + v];
    for (int u = 0; u < w; ++u) s = decayed(s_l[u][lane][v], s) + s_h[u][lane][v];
#pragma unroll
    for (int k = 0; k < T; ++k) {
      before[k][v] = s;
      s = fmaf(a[k][v], s, b[k][v]);
    }
  }
  float q_sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) q_sum[v] = 0.f;
#pragma unroll
  for (int k = T - 1; k >= 0; --k) {
    if (t0 + k >= g.L) continue;
    const long long at = (row0 + t0 + k) * g.ld_out + ch;
    Lane<E, V> ox, oi, oR, oz;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float xx = to_f(x[k].v[v]), gate = sigmoid_exact(to_f(in[k].v[v])), open = sigmoid_exact(to_f(r[k].v[v]));
      const float l = rate[v] * open;
      float aa, m;
      decay_of(l, aa, m);
      const float G = upstream(k, v) + carry[v];
      if (g.z != nullptr) {
        const float zz = to_f(z[k].v[v]), s = sigmoid_exact(zz);
        oz.v[v] = from_f<E>(to_f(gy[k].v[v]) * fmaf(aa, before[k][v], b[k][v]) * s * (1.f + zz * (1.f - s)));
      }
      const float gm = G * m * gate;
      ox.v[v] = from_f<E>(gm);
      oi.v[v] = from_f<E>(gm * xx * (1.f - gate));
      const float back = m > 0.f ? aa * aa * -l * __builtin_amdgcn_rcpf(m) : 0.f;
      const float q = G * fmaf(aa * l, before[k][v], gate * xx * back);
      oR.v[v] = from_f<E>(q * (1.f - open));
      q_sum[v] += q;
      carry[v] = aa * G;
    }
    if (active) {
      if (g.gx != nullptr) *reinterpret_cast<Lane<E, V>*>(g.gx + at) = ox;
      if (g.gi != nullptr) *reinterpret_cast<Lane<E, V>*>(g.gi + at) = oi;
      if (g.gr != nullptr) *reinterpret_cast<Lane<E, V>*>(g.gr + at) = oR;
      if (g.gz != nullptr) *reinterpret_cast<Lane<E, V>*>(g.gz + at) = oz;
    }
  }
  if (c == 0 && w == 0 && active && g.gstart != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) g.gstart[static_cast<size_t>(seq) * g.D + ch + v] = carry[v];
  }
  if (g.partial == nullptr) return;
  __syncthreads();  // the states' aggregates are read
#pragma unroll
  for (int v = 0; v < V; ++v) s_h[w][lane][v] = q_sum[v];
  __syncthreads();
  if (w == 0 && active) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float t = 0.f;
#pragma unroll
      for (int u = 0; u < W; ++u) t += s_h[u][lane][v];
      g.partial[(static_cast<size_t>(c) * g.B + seq) * g.D + ch + v] = t;
    }
  }
}

// ---- single tokens ------------------------------------------------------------------------
template <class E, int V>
__global__ __launch_bounds__(256) void recurrence_step_kernel(Forward<E> g) {
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int lanes = g.D / V;
  const long long row = at / lanes;
  if (row >= g.L) return;
  const int ch = static_cast<int>(at - row * lanes) * V;
  const int from = g.slots[row], to = g.out_slots[row];
  const bool have = from >= 0 && from < g.n_slots, keep = to >= 0 && to < g.n_slots;
  const Lane<E, V> r = lane_load<E, V>(g.r + row * g.ld_r + ch), in = lane_load<E, V>(g.i + row * g.ld_i + ch),
                   x = lane_load<E, V>(g.x + row * g.ld_x + ch);
  Lane<E, V> z{}, out;
  if (g.z != nullptr) z = lane_load<E, V>(g.z + row * g.ld_z + ch);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float a, m;
    const float l = -decay_rate(g.decay[ch + v], g.scale) * sigmoid_exact(to_f(r.v[v]));
    decay_of(l, a, m);
    float h = m * sigmoid_exact(to_f(in.v[v])) * to_f(x.v[v]);
    if (have) h = fmaf(a, g.pool[static_cast<size_t>(from) * g.D + ch + v], h);
    if (keep) g.pool[static_cast<size_t>(to) * g.D + ch + v] = h;
    if (g.z != nullptr) {
      const float zz = to_f(z.v[v]);
      h *= zz * sigmoid_exact(zz);
    }
    out.v[v] = from_f<E>(have || keep ? h : 0.f);
  }
  *reinterpret_cast<Lane<E, V>*>(g.y + row * g.D + ch) = out;
}

// ---- launches -----------------------------------------------------------------------------
int64_t chunks_of(int64_t L, int waves) { return L > 0 ? (L + kSteps * waves - 1) / (kSteps * waves) : 1; }

// Two channels a lane of 16-bit elements where every row lies on whole words.
template <class E>
bool in_pairs(int64_t D, std::initializer_list<int64_t> strides, std::initializer_list<const void*> ps) {
  if (sizeof(E) != 2 || D % 2 != 0) return false;
  for (int64_t s : strides)
    if (s % 2 != 0) return false;
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return false;
  return true;
}

template <class E, int V, bool PACKED>
int forward_v(Forward<E> g, StreamCall& call) {
  const char* what = PACKED ? "recurrence_prompt" : "recurrence_forward";
  g.n_cols = (g.D + 64 * V - 1) / (64 * V);
  const int64_t groups = int64_t(g.B) * g.n_cols, total = groups * g.n_chunks;
  if (int rc = check_grid(what, total, kWaves * 64)) return rc;
  void* records = nullptr;
  LaunchSync sync{};
  if (int rc = acquire_scratch(call, static_cast<size_t>(total) * kRecords * 64 * V * 8, total, &records, &sync)) return rc;
  hipLaunchKernelGGL((recurrence_forward_kernel<E, V, kSteps, kWaves, PACKED>), dim3(static_cast<unsigned>(total)),
                     dim3(kWaves * 64), 0, call.stream(), g, static_cast<unsigned long long*>(records), sync);
  return launch_check("recurrence_forward_kernel");
}

template <class E, bool PACKED>
int forward(Forward<E> g, StreamCall& call) {
  const bool pairs = in_pairs<E>(g.D, {g.ld_x, g.ld_i, g.ld_r, g.z ? g.ld_z : 0}, {g.x, g.i, g.r, g.z, g.y});
  if constexpr (sizeof(E) == 2)
    if (pairs) return forward_v<E, 2, PACKED>(g, call);
  return forward_v<E, 1, PACKED>(g, call);
}

template <class E, int V>
int backward_v(Backward<E> g, float* gdecay, StreamCall& call) {
  const char* what = "recurrence_backward";
  g.n_cols = (g.D + 64 * V - 1) / (64 * V);
  const int64_t groups = int64_t(g.B) * g.n_cols, total = groups * g.n_chunks;
  if (int rc = check_grid(what, total, kBackWaves * 64)) return rc;
  if (gdecay != nullptr) {
    void* p = nullptr;
    if (int rc = acquire_workspace(call, static_cast<size_t>(g.n_chunks) * g.B * g.D * sizeof(float), &p)) return rc;
    g.partial = static_cast<float*>(p);
  }
  void* records = nullptr;
  LaunchSync sync{};
  if (int rc = acquire_scratch(call, static_cast<size_t>(total) * kRecords * 64 * V * 8, total, &records, &sync)) return rc;
  hipLaunchKernelGGL((recurrence_backward_kernel<E, V, kSteps, kBackWaves>), dim3(static_cast<unsigned>(total)),
                     dim3(kBackWaves * 64), 0, call.stream(), g, static_cast<unsigned long long*>(records), sync);
  if (int rc = launch_check("recurrence_backward_kernel")) return rc;
  if (gdecay == nullptr) return OSSM_OK;
  hipLaunchKernelGGL(decay_grad_kernel, dim3(static_cast<unsigned>((g.D + 63) / 64)), dim3(1024), 0, call.stream(), g.partial,
                     g.n_chunks * g.B, g.D, g.decay, gdecay);
  return launch_check("decay_grad_kernel");
}

int check_sizes(const char* what, int dtype, int64_t B, int64_t L, int64_t D) {
  if (dtype != OSSM_F32 && dtype != OSSM_BF16)
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": unknown dtype");
  if (B < 0 || L < 0 || D < 0) return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  if (B > (1 << 24) || L > (1 << 30) || D > (1 << 24))
    return set_error(OSSM_ERR_UNSUPPORTED, std::string(what) + ": size exceeds launch limits");
  return OSSM_OK;
}

int null_pointer(const char* what) { return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": null pointer"); }

int short_rows(const char* what) {
  return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": row stride below the row");
}

}  // namespace
}  // namespace ossm

using namespace ossm;

extern "C" {

int64_t ossm_recurrence_saved(int64_t batch, int64_t length, int64_t dim) {
  return batch * chunks_of(length, kBackWaves) * dim;
}

int ossm_recurrence_forward(int dtype, const void* x, int64_t ld_x, const void* input_gate, int64_t ld_input_gate,
                            const void* decay_gate, int64_t ld_decay_gate, const void* output_gate, int64_t ld_output_gate,
                            const float* decay, float scale, const float* start, void* y, float* last, float* saved,
                            int64_t batch, int64_t length, int64_t dim, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "recurrence_forward";
  if (int rc = check_sizes(what, dtype, batch, length, dim)) return rc;
  if (batch == 0 || length == 0 || dim == 0) return OSSM_OK;
  if (!x || !input_gate || !decay_gate || !decay || !y || !last) return null_pointer(what);
  if (batch * length > 1 && (ld_x < dim || ld_input_gate < dim || ld_decay_gate < dim || (output_gate && ld_output_gate < dim)))
    return short_rows(what);
  StreamCall call(static_cast<hipStream_t>(stream_v));
  if (call.status()) return call.status();
  const auto go = [&](auto e) {
    using E = decltype(e);
    Forward<E> g{};
    g.x = static_cast<const E*>(x), g.ld_x = ld_x;
    g.i = static_cast<const E*>(input_gate), g.ld_i = ld_input_gate;
    g.r = static_cast<const E*>(decay_gate), g.ld_r = ld_decay_gate;
    g.z = static_cast<const E*>(output_gate), g.ld_z = ld_output_gate;
    g.decay = decay, g.scale = scale, g.start = start;
    g.y = static_cast<E*>(y), g.last = last, g.saved = saved;
    g.B = static_cast<int>(batch), g.L = static_cast<int>(length), g.D = static_cast<int>(dim);
    g.n_chunks = static_cast<int>(chunks_of(length, kWaves));
    g.n_saved = static_cast<int>(chunks_of(length, kBackWaves));
    return forward<E, false>(g, call);
  };
  return dtype == OSSM_BF16 ? go(bf16_t{}) : go(0.f);
}

int ossm_recurrence_backward(int dtype, const void* grad_y, int64_t ld_grad, const float* grad_last, const void* x, int64_t ld_x,
                             const void* input_gate, int64_t ld_input_gate, const void* decay_gate, int64_t ld_decay_gate,
                             const void* output_gate, int64_t ld_output_gate, const float* decay, float scale,
                             const float* saved, void* grad_x, void* grad_input_gate, void* grad_decay_gate,
                             void* grad_output_gate, int64_t ld_grads, float* grad_decay, float* grad_start, int64_t batch,
                             int64_t length, int64_t dim, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "recurrence_backward";
  if (int rc = check_sizes(what, dtype, batch, length, dim)) return rc;
  if (batch == 0 || length == 0 || dim == 0) return OSSM_OK;
  if (!grad_y || !x || !input_gate || !decay_gate || !decay || !saved || (grad_output_gate && !output_gate))
    return null_pointer(what);
  if (batch * length > 1 && (ld_grad < dim || ld_grads < dim || ld_x < dim || ld_input_gate < dim || ld_decay_gate < dim ||
                             (output_gate && ld_output_gate < dim)))
    return short_rows(what);
  StreamCall call(static_cast<hipStream_t>(stream_v));
  if (call.status()) return call.status();
  const auto go = [&](auto e) {
    using E = decltype(e);
    Backward<E> g{};
    g.x = static_cast<const E*>(x), g.ld_x = ld_x;
    g.i = static_cast<const E*>(input_gate), g.ld_i = ld_input_gate;
    g.r = static_cast<const E*>(decay_gate), g.ld_r = ld_decay_gate;
    g.z = static_cast<const E*>(output_gate), g.ld_z = ld_output_gate;
    g.gy = static_cast<const E*>(grad_y), g.ld_gy = ld_grad;
    g.decay = decay, g.scale = scale, g.saved = saved, g.glast = grad_last;
    g.gx = static_cast<E*>(grad_x), g.gi = static_cast<E*>(grad_input_gate), g.gr = static_cast<E*>(grad_decay_gate);
    g.gz = static_cast<E*>(grad_output_gate), g.ld_out = ld_grads, g.gstart = grad_start;
    g.B = static_cast<int>(batch), g.L = static_cast<int>(length), g.D = static_cast<int>(dim);
    g.n_chunks = static_cast<int>(chunks_of(length, kBackWaves));
    const bool pairs = in_pairs<E>(dim, {ld_x, ld_input_gate, ld_decay_gate, output_gate ? ld_output_gate : 0, ld_grad, ld_grads},
                                   {x, input_gate, decay_gate, output_gate, grad_y, grad_x, grad_input_gate, grad_decay_gate,
                                    grad_output_gate});
    if constexpr (sizeof(E) == 2)
      if (pairs) return backward_v<E, 2>(g, grad_decay, call);
    return backward_v<E, 1>(g, grad_decay, call);
  };
  return dtype == OSSM_BF16 ? go(bf16_t{}) : go(0.f);
}

int ossm_recurrence_prompt(int dtype, const void* x, int64_t ld_x, const void* input_gate, int64_t ld_input_gate,
                           const void* decay_gate, int64_t ld_decay_gate, const void* output_gate, int64_t ld_output_gate,
                           const float* decay, float scale, float* state, const int32_t* in_slots, const int32_t* out_slots,
                           const int32_t* offsets, const uint8_t* resume, void* y, int64_t rows, int64_t n_seqs,
                           int64_t n_slots, int64_t dim, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "recurrence_prompt";
  if (int rc = check_sizes(what, dtype, n_seqs, rows, dim)) return rc;
  if (n_slots < 0 || n_slots > INT_MAX) return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": bad pool size");
  if (n_seqs > 65535) return set_error(OSSM_ERR_UNSUPPORTED, std::string(what) + ": more than 65535 prompts");
  if (dim == 0 || (rows == 0 && n_seqs == 0)) return OSSM_OK;
  if ((rows > 0 && (!x || !input_gate || !decay_gate || !y)) || !decay || (n_seqs > 0 && (!in_slots || !offsets)) ||
      (n_slots > 0 && !state))
    return null_pointer(what);
  if (rows > 1 && (ld_x < dim || ld_input_gate < dim || ld_decay_gate < dim || (output_gate && ld_output_gate < dim)))
    return short_rows(what);
  StreamCall call(static_cast<hipStream_t>(stream_v));
  if (call.status()) return call.status();
  const auto go = [&](auto e) {
    using E = decltype(e);
    Forward<E> g{};
    g.x = static_cast<const E*>(x), g.ld_x = ld_x;
    g.i = static_cast<const E*>(input_gate), g.ld_i = ld_input_gate;
    g.r = static_cast<const E*>(decay_gate), g.ld_r = ld_decay_gate;
    g.z = static_cast<const E*>(output_gate), g.ld_z = ld_output_gate;
    g.decay = decay, g.scale = scale, g.y = static_cast<E*>(y);
    g.pool = state, g.slots = in_slots, g.out_slots = out_slots ? out_slots : in_slots;
    g.offsets = offsets, g.resume = resume;
    g.n_seqs = static_cast<int>(n_seqs), g.n_slots = static_cast<int>(n_slots);
    g.B = 1, g.L = static_cast<int>(rows), g.D = static_cast<int>(dim);
    g.n_chunks = static_cast<int>(chunks_of(rows, kWaves));
    return forward<E, true>(g, call);
  };
  return dtype == OSSM_BF16 ? go(bf16_t{}) : go(0.f);
}

int ossm_recurrence_step(int dtype, const void* x, int64_t ld_x, const void* input_gate, int64_t ld_input_gate,
                         const void* decay_gate, int64_t ld_decay_gate, const void* output_gate, int64_t ld_output_gate,
                         const float* decay, float scale, float* state, const int32_t* in_slots, const int32_t* out_slots,
                         void* y, int64_t rows, int64_t n_slots, int64_t dim, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "recurrence_step";
  if (int rc = check_sizes(what, dtype, 1, rows, dim)) return rc;
  if (n_slots < 0 || n_slots > INT_MAX) return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": bad pool size");
  if (dim == 0 || rows == 0) return OSSM_OK;
  if (!x || !input_gate || !decay_gate || !y || !decay || !in_slots || (n_slots > 0 && !state)) return null_pointer(what);
  if (rows > 1 && (ld_x < dim || ld_input_gate < dim || ld_decay_gate < dim || (output_gate && ld_output_gate < dim)))
    return short_rows(what);
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  const auto go = [&](auto e) {
    using E = decltype(e);
    Forward<E> g{};
    g.x = static_cast<const E*>(x), g.ld_x = ld_x;
    g.i = static_cast<const E*>(input_gate), g.ld_i = ld_input_gate;
    g.r = static_cast<const E*>(decay_gate), g.ld_r = ld_decay_gate;
    g.z = static_cast<const E*>(output_gate), g.ld_z = ld_output_gate;
    g.decay = decay, g.scale = scale, g.y = static_cast<E*>(y);
    g.pool = state, g.slots = in_slots, g.out_slots = out_slots ? out_slots : in_slots;
    g.n_slots = static_cast<int>(n_slots), g.L = static_cast<int>(rows), g.D = static_cast<int>(dim);
    const bool pairs = in_pairs<E>(dim, {ld_x, ld_input_gate, ld_decay_gate, output_gate ? ld_output_gate : 0},
                                   {x, input_gate, decay_gate, output_gate, y});
    const int64_t groups = (rows * (pairs ? dim / 2 : dim) + 255) / 256;
    if (int rc = check_grid(what, groups, 256)) return rc;
    if constexpr (sizeof(E) == 2)
      if (pairs) {
        hipLaunchKernelGGL((recurrence_step_kernel<E, 2>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, g);
        return launch_check("recurrence_step_kernel");
      }
    hipLaunchKernelGGL((recurrence_step_kernel<E, 1>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, g);
    return launch_check("recurrence_step_kernel");
  };
  return dtype == OSSM_BF16 ? go(bf16_t{}) : go(0.f);
}

}  // extern "C"
