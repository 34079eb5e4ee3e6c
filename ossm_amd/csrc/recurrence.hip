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
//   q = l dL/dl = a G l (h_{t-1} - a b / (1 - a^2)),   gr = q (1 - sigmoid(r)),   b = m g x
//   gdecay = sigmoid(decay) / softplus(decay) sum of q
//
// It is bound by memory, with the operations close behind: [4, 8192, 2048] in bf16 with a gate takes
// 165 us forward, of which 134 are its bytes' at a copy's rate and 93 (57 percent of the cycles) VALU
// issue; 301 backward, 242 and 160.  So each tensor is read once: time is cut into chunks
// of T W steps, a workgroup of W waves takes a chunk of 64 V channels (V a lane),
// wave w its steps from w T on.  Each wave folds its steps into
// one (sum of l, state from zero), the waves are joined through LDS, and the chunk's start comes
// from the chunks before it by records in the stream's scratch.  A chunk's place among P
// neighbours is fixed: it waits for the aggregates of its neighbours before it and for the state
// at the end of the P before them, so the wait is one round trip for P chunks, and
// every sum has one order: results are bitwise repeatable.
//
// l is kept to base 2, so that a is one instruction's result.  Decays over several steps are
// kept as sums of l and applied in two halves: exp(l) of a
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

constexpr int kSavedEvery = 32;  // steps between the states that the forward saves for the backward

constexpr float kTiny = 1.17549435e-38f;  // the smallest normal number

// ---- the step's values ----------------------------------------------------------
// NaN passes through the greatest of two, which fmaxf would drop.
__device__ __forceinline__ float greatest(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// kFull: float32's inputs and outputs.  x log2(e) is rounded, which costs the exponential
// |x| 2^-24 of itself; kFull puts the rest back (four operations of some forty).  16-bit
// inputs are sums of products rounded to 2^-9 of themselves, at which 2^-22 is no loss.
// The reciprocal is the hardware's, within 1 ulp.
template <bool kFull>
__device__ __forceinline__ float sigmoid_of(float x) {
  constexpr float kLog2e = 1.44269504f, kRest = 1.92596299e-8f, kLn2 = 0.693147181f;
  float e;
  if constexpr (kFull) {
    const float b = __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, 88.f), -88.f);  // no inf - inf
    const float y = -kLog2e * b;
    e = __builtin_amdgcn_exp2f(y);
    e = fmaf(e, kLn2 * fmaf(-kRest, b, fmaf(-kLog2e, b, -y)), e);
  } else {
    e = __builtin_amdgcn_exp2f(-kLog2e * x);
  }
  return __builtin_amdgcn_rcpf(1.f + e);
}

// a = 2^l and 1 - a^2 of a log-decay l <= 0 (to base 2).  a is no less than the smallest normal
// number, by which an infinite state stays infinite: a step leaves at least 2^-126 of a state.
// Near zero 1 - a^2 is the series of -expm1 (what is left out is below 2^-24 of it); from where
// a^2 is far enough from one it is 1 - a a, at 0.67 with three times a's rounding, in 16 bits at
// 0.88 with eight.
template <bool kFull>
__device__ __forceinline__ void decay_of(float l, float& a, float& rest) {
  a = greatest(__builtin_amdgcn_exp2f(l), kTiny);
  // -(2 ln 2)^n / n!
  float s;
  if constexpr (kFull) {
    s = -0.00195234993f;
    s = fmaf(s, l, -0.00985825945f);
    s = fmaf(s, l, -0.0426673861f);
  } else {
    s = -0.0426673861f;
  }
  s = fmaf(s, l, -0.153890066f);
  s = fmaf(s, l, -0.444032869f);
  s = fmaf(s, l, -0.960906028f);
  s = fmaf(s, l, -1.38629436f);
  rest = l > (kFull ? -0.29f : -0.09f) ? s * l : fmaf(-a, a, 1.f);
}

// A decay over several steps, 2^l, as the half of it that is applied twice.  -inf is zero:
// nothing before counts, whatever it holds.
__device__ __forceinline__ float half_of(float l) {
  return l == -__builtin_inff() ? 0.f : greatest(__builtin_amdgcn_exp2f(0.5f * l), kTiny);
}
__device__ __forceinline__ float decayed(float half, float h) { return half == 0.f ? 0.f : (h * half) * half; }

// scale softplus(decay), to base 2: -log2 of the decay at a gate wide open.  softplus(x) =
// max(x, 0) + log1p(e), e = exp(-|x|), the logarithm by its series in z = e / (2 + e) <= 1/3 as
// softplus_f's, of an exponential that keeps its digits at any x.
__device__ __forceinline__ float decay_rate(float decay, float scale) {
  constexpr float kLog2e = 1.44269504f, kRest = 1.92596299e-8f, kLn2 = 0.693147181f;
  const float x = fabsf(decay), y = -kLog2e * x;
  float e = __builtin_amdgcn_exp2f(y);
  e = x < 88.f ? fmaf(e, kLn2 * fmaf(-kRest, x, fmaf(-kLog2e, x, -y)), e) : e;
  const float z = e * __builtin_amdgcn_rcpf(2.f + e), q = z * z;
  float s = 1.f / 15.f;
  s = fmaf(s, q, 1.f / 13.f);
  s = fmaf(s, q, 1.f / 11.f);
  s = fmaf(s, q, 1.f / 9.f);
  s = fmaf(s, q, 1.f / 7.f);
  s = fmaf(s, q, 1.f / 5.f);
  s = fmaf(s, q, 1.f / 3.f);
  s = fmaf(s, q, 1.f);
  return kLog2e * scale * (greatest(decay, 0.f) + 2.f * z * s);
}

// gdecay from the chunks' sums of q; 7 us at [4, 8192, 2048], 1024 sums a channel.
__global__ __launch_bounds__(kSumThreads) void decay_grad_kernel(const float* partial, int n, int D, const float* decay, float* out) {
  const double t = column_sum(partial, n, D, D);
  const int i = static_cast<int>(blockIdx.x) * kSumColumns + threadIdx.x;
  if (threadIdx.x >= kSumColumns || i >= D) return;
  const double x = decay[i];
  // sigmoid / softplus goes to one below; past -40 the quotient's own terms vanish
  const double ratio = x < -40 ? 1. : 1. / ((1. + exp(-x)) * (fmax(x, 0.) + log1p(exp(-fabs(x)))));
  out[i] = static_cast<float>(t * ratio);
}

// A quotient that is the same in every lane, as a scalar: rows' addresses then are scalars too.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---- records ------------------------------------------------------------------------
// Per chunk and channel: the aggregate's sum of l and state, and the state at the
// chunk's end (written by the last chunk of P neighbours only).
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

// Waits for the V tagged words at each of the first n of p and q (the same may be given twice);
// NaN where the wait gives up.  All are asked for at once: one round trip, not n.
template <int V, int R>
__device__ __forceinline__ void await(const unsigned long long* const (&p)[R], const unsigned long long* const (&q)[R], int n,
                                      const LaunchSync& sync, float (&vp)[R][V], float (&vq)[R][V]) {
  bool done = sync.poison != 0;
  for (uint32_t spins = 0; !done; ++spins) {
    unsigned long long a[R][V], b[R][V];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= n) break;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        a[i][k] = __hip_atomic_load(p[i] + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        b[i][k] = __hip_atomic_load(q[i] + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    bool ok = true;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= n) break;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        ok = ok && static_cast<unsigned>(a[i][k] >> 32) == sync.tag && static_cast<unsigned>(b[i][k] >> 32) == sync.tag;
        vp[i][k] = __uint_as_float(static_cast<unsigned>(a[i][k]));
        vq[i][k] = __uint_as_float(static_cast<unsigned>(b[i][k]));
      }
    }
    if (ok) return;
    if (spins > kSpinLimit) {
      __hip_atomic_fetch_or(sync.err, kErrSpinTimeout, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      done = true;
    }
    __builtin_amdgcn_s_sleep(1);
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) vp[i][k] = vq[i][k] = __builtin_nanf("");
}

// One workgroup's part of the scan between chunks.
template <int V, int W, int P>
struct Join {
  float l[W][64][V], half[W][64][V], h[W][64][V];   // the waves' aggregates: sum of l, its half, state from zero
  float before[P][64][V], state[P][64][V];  // those of the neighbours before: half, state
  float carry[64][V];
};

// Two stretches' halves as one's; neither a reset nor an infinite state's decay is lost.
__device__ __forceinline__ float joined(float p, float q) { return p == 0.f || q == 0.f ? 0.f : greatest(p * q, kTiny); }

// j: the chunk's place in the scan's order (in the backward counted from the end); w: the
// calling wave's, l and h its aggregate; start: the state before the first chunk.  Gives the
// state from which the calling wave starts.
template <int V, int W, int P>
__device__ __forceinline__ void join_chunks(Join<V, W, P>& s, int w, int lane, int j, int n_chunks, const Rec& rec, size_t ch,
                                            const LaunchSync& sync, float (&l)[V], float (&h)[V], const float (&start)[V],
                                            float (&carry)[V]) {
  const int place = j % P;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    s.l[w][lane][k] = l[k];
    s.half[w][lane][k] = half_of(l[k]);
    s.h[w][lane][k] = h[k];
  }
  __syncthreads();
  const bool more = j + 1 < n_chunks;
  if (more && place + 1 < P && w == W - 1) {  // the chunk's aggregate, for its neighbours
    float al[V], ah[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      al[k] = s.l[0][lane][k];
      ah[k] = s.h[0][lane][k];
#pragma unroll
      for (int v = 1; v < W; ++v) {
        const float d = s.l[v][lane][k];
        ah[k] = decayed(s.half[v][lane][k], ah[k]) + s.h[v][lane][k];
        al[k] = d == -__builtin_inff() ? d : al[k] + d;
      }
    }
    publish<V>(rec.at(j, kSumL, ch), al, sync.tag);
    publish<V>(rec.at(j, kState, ch), ah, sync.tag);
  }
  constexpr int R = P / W;  // neighbours a wave waits for: w R and on
  if (w * R < place) {
    const unsigned long long* p[R];
    const unsigned long long* q[R];
    float a[R][V], b[R][V];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      p[i] = rec.at(j - place + w * R + i, kSumL, ch);
      q[i] = rec.at(j - place + w * R + i, kState, ch);
    }
    await<V, R>(p, q, place - w * R, sync, a, b);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (w * R + i >= place) break;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        s.before[w * R + i][lane][k] = half_of(a[i][k]);
        s.state[w * R + i][lane][k] = b[i][k];
      }
    }
  }
  // what the waves before do to the chunk's start
  float wave_half[V], wave_h[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    wave_half[k] = 1.f;
    wave_h[k] = 0.f;
    for (int v = 0; v < w; ++v) {
      const float d = s.half[v][lane][k];
      wave_half[k] = joined(wave_half[k], d);
      wave_h[k] = decayed(d, wave_h[k]) + s.h[v][lane][k];
    }
  }
  if (place > 0) __syncthreads();
  if (w == W - 1) {
    // all that is known before the neighbours' own start arrives, so that it is passed on at once
    float half[V], state[V], end_half[V], end_h[V], first[1][V], unused[1][V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      half[k] = 1.f;
      state[k] = 0.f;
      for (int v = 0; v < place; ++v) {
        const float d = s.before[v][lane][k];
        half[k] = joined(half[k], d);
        state[k] = decayed(d, state[k]) + s.state[v][lane][k];
      }
      const float d = s.half[w][lane][k];
      end_half[k] = joined(wave_half[k], d);
      end_h[k] = decayed(d, wave_h[k]) + h[k];
      first[0][k] = start[k];
    }
    if (j > place) {
      const unsigned long long* const p[1] = {rec.at(j - place - 1, kEnd, ch)};
      await<V, 1>(p, p, 1, sync, first, unused);
    }
    float end[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float c = decayed(half[k], first[0][k]) + state[k];
      s.carry[lane][k] = c;
      end[k] = decayed(end_half[k], c) + end_h[k];
    }
    if (more && place == P - 1) publish<V>(rec.at(j, kEnd, ch), end, sync.tag);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < V; ++k) carry[k] = decayed(wave_half[k], s.carry[lane][k]) + wave_h[k];
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
  float* saved;  // [B, n_saved, D] the state before every kSavedEvery steps, or null
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
__device__ __forceinline__ Lane<E, V> lane_load(const E* row, unsigned ch) {
  return *reinterpret_cast<const Lane<E, V>*>(row + ch);
}
template <class E, int V>
__device__ __forceinline__ void lane_store(E* row, unsigned ch, const Lane<E, V>& v) {
  // past the caches: written once, read by later kernels only
  if constexpr (V * sizeof(E) == 4) __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, v), reinterpret_cast<uint32_t*>(row + ch));
  else __builtin_nontemporal_store(__builtin_bit_cast(uint16_t, v), reinterpret_cast<uint16_t*>(row + ch));
}

// h of a prompt before its first token
template <class E, int V>
__device__ __forceinline__ void prompt_start(const Forward<E>& g, int seq, unsigned ch, float (&h)[V]) {
  const int slot = g.resume != nullptr && g.resume[seq] ? g.slots[seq] : -1;
#pragma unroll
  for (int k = 0; k < V; ++k)
    h[k] = slot >= 0 && slot < g.n_slots ? g.pool[static_cast<size_t>(slot) * g.D + ch + k] : 0.f;
}

template <class E, int V>
__device__ __forceinline__ void prompt_end(const Forward<E>& g, int seq, unsigned ch, bool active, const float (&h)[V]) {
  const int slot = g.out_slots[seq];
  if (!active || slot < 0 || slot >= g.n_slots) return;
#pragma unroll
  for (int k = 0; k < V; ++k) g.pool[static_cast<size_t>(slot) * g.D + ch + k] = h[k];
}

template <class E, int V, int T, int W, int P, bool PACKED, bool GATE>
__global__ __launch_bounds__(W * 64) void recurrence_forward_kernel(Forward<E> g, unsigned long long* records, LaunchSync sync) {
  constexpr bool kFull = sizeof(E) == 4;
  __shared__ Join<V, W, P> s_join;
  __shared__ int s_first[PACKED ? T * W : 1], s_final[PACKED ? T * W : 1];  // the prompt that starts, ends at a token, + 1
  __shared__ int s_ticket;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int n_groups = g.B * g.n_cols;
  const int ticket = launch_order(sync, n_groups * g.n_chunks, &s_ticket);
  const int c = uniform(ticket / n_groups), group = ticket - c * n_groups;
  const int seq = uniform(group / g.n_cols), col = group - seq * g.n_cols;
  const unsigned ch_raw = static_cast<unsigned>(col * 64 + lane) * V;
  const bool active = ch_raw < static_cast<unsigned>(g.D);
  const unsigned ch = active ? ch_raw : g.D - V;  // past the end: the last channels, never stored
  const int t_chunk = c * T * W, t0 = t_chunk + w * T;
  const long long row0 = static_cast<long long>(seq) * g.L;

  // everything is asked for before anything is used, in the order of use
  float rate[V];
#pragma unroll
  for (int k = 0; k < V; ++k) rate[k] = g.decay[ch + k];
  Lane<E, V> x[T], in[T], r[T], z[T];
  // Without a condition, also for prompts of no rows, which load some row and use nothing of it:
  // behind one, 16-bit elements are held one a register (168 of them against 120, 3 waves a SIMD).
  const auto row_of = [&](int k) {
    const int t = min(t0 + k, g.L - 1);
    return row0 + (PACKED ? max(t, 0) : t);
  };
#pragma unroll
  for (int k = 0; k < T; ++k) {
    r[k] = lane_load<E, V>(g.r + row_of(k) * g.ld_r, ch);
    in[k] = lane_load<E, V>(g.i + row_of(k) * g.ld_i, ch);
    x[k] = lane_load<E, V>(g.x + row_of(k) * g.ld_x, ch);
  }
#pragma unroll
  for (int k = 0; k < T; ++k)
    if (GATE) z[k] = lane_load<E, V>(g.z + row_of(k) * g.ld_z, ch);
  const int lo = PACKED && g.n_seqs > 0 ? g.offsets[0] : 0, hi = PACKED && g.n_seqs > 0 ? g.offsets[g.n_seqs] : 0;
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (PACKED) {
    for (int k = threadIdx.x; k < T * W; k += W * 64) s_first[k] = s_final[k] = 0;
    __syncthreads();
    // a stretch of prompts a thread: only one whose tokens meet the chunk's is looked through
    const int span = (g.n_seqs + W * 64 - 1) / (W * 64), s0 = min(static_cast<int>(threadIdx.x) * span, g.n_seqs);
    const int s1 = min(s0 + span, g.n_seqs);
    if (s0 < s1 && g.offsets[s0] < t_chunk + T * W && g.offsets[s1] >= t_chunk) {
      for (int s = s0; s < s1; ++s) {
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
  float a[T][V], b[T][V], sum[V], h[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    rate[k] = -decay_rate(rate[k], g.scale);
    sum[k] = h[k] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < T; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // past the end l is zero, and the state stays
      const float l = t0 + k < g.L ? rate[v] * sigmoid_of<kFull>(to_f(r[k].v[v])) : 0.f;
      float rest;
      decay_of<kFull>(l, a[k][v], rest);
      b[k][v] = __builtin_amdgcn_sqrtf(rest) * (sigmoid_of<kFull>(to_f(in[k].v[v])) * to_f(x[k].v[v]));
      sum[v] += l;
      h[v] = fmaf(a[k][v], h[v], b[k][v]);
    }
  }
  // which of the wave's tokens start and end a prompt
  const unsigned long long firsts = PACKED ? __ballot(lane < T && s_first[w * T + lane % T] != 0) : 0;
  const unsigned long long finals = PACKED ? __ballot(lane < T && s_final[w * T + lane % T] != 0) : 0;
  if (firsts != 0) {
    // apart from the loop above: a branch at each of its steps cost 4 percent of a long batch
#pragma unroll
    for (int k = 0; k < T; ++k) {
      if (firsts >> k & 1) {
        float init[V];
        prompt_start<E, V>(g, __builtin_amdgcn_readfirstlane(s_first[w * T + k]) - 1, ch, init);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = b[k][v] = fmaf(a[k][v], init[v], b[k][v]);
          a[k][v] = -1.f;  // nothing before counts
          sum[v] = -__builtin_inff();
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(a[k][v], h[v], b[k][v]);
      }
    }
  }
  const Rec rec{records, static_cast<size_t>(n_groups) * 64 * V};
  const size_t rec_ch = (static_cast<size_t>(group) * 64 + lane) * V;
  float start[V], carry[V];
#pragma unroll
  for (int k = 0; k < V; ++k) start[k] = !PACKED && g.start != nullptr ? g.start[static_cast<size_t>(seq) * g.D + ch + k] : 0.f;
  join_chunks<V, W, P>(s_join, w, lane, c, g.n_chunks, rec, rec_ch, sync, sum, h, start, carry);

  if (!PACKED && g.saved != nullptr && t0 % kSavedEvery == 0 && t0 < g.L && active) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      g.saved[(static_cast<size_t>(seq) * g.n_saved + t0 / kSavedEvery) * g.D + ch + k] = carry[k];
  }
#pragma unroll
  for (int k = 0; k < T; ++k) {
    if (t0 + k >= g.L) break;
    Lane<E, V> out;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      carry[v] = PACKED && a[k][v] < 0.f ? b[k][v] : fmaf(a[k][v], carry[v], b[k][v]);
      float y = carry[v];
      if (GATE) {
        const float zz = to_f(z[k].v[v]);
        y *= zz * sigmoid_of<kFull>(zz);
      }
      if (PACKED && (t0 + k < lo || t0 + k >= hi)) y = 0.f;
      out.v[v] = from_f<E>(y);
    }
    if (active) lane_store<E, V>(g.y + (row0 + t0 + k) * g.D, ch, out);
    if constexpr (PACKED) {
      if (finals >> k & 1) prompt_end<E, V>(g, __builtin_amdgcn_readfirstlane(s_final[w * T + k]) - 1, ch, active, carry);
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
  const float* saved;  // [B, n_saved, D]
  const float* glast;  // [B, D] or null
  E* gx;
  E* gi;
  E* gr;
  E* gz;
  float* gstart;   // [B, D] or null
  float* partial;  // [n_chunks B, D] sums of q
  int B, L, D, n_cols, n_chunks, n_saved;
};

template <class E, int V, int T, int W, int P, bool GATE>
__global__ __launch_bounds__(W * 64) void recurrence_backward_kernel(Backward<E> g, unsigned long long* records, LaunchSync sync) {
  constexpr bool kFull = sizeof(E) == 4;
  constexpr float kLn2 = 0.693147181f;
  __shared__ Join<V, W, P> s_join;
  __shared__ float s_l[W][64][V], s_h[W][64][V];
  __shared__ int s_ticket;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int n_groups = g.B * g.n_cols;
  const int ticket = launch_order(sync, n_groups * g.n_chunks, &s_ticket);
  const int j = uniform(ticket / n_groups), group = ticket - j * n_groups;
  const int c = g.n_chunks - 1 - j;  // the last chunk first
  const int seq = uniform(group / g.n_cols), col = group - seq * g.n_cols;
  const unsigned ch_raw = static_cast<unsigned>(col * 64 + lane) * V;
  const bool active = ch_raw < static_cast<unsigned>(g.D);
  const unsigned ch = active ? ch_raw : g.D - V;
  const int t0 = c * T * W + w * T;
  const long long row0 = static_cast<long long>(seq) * g.L;

  float rate[V], first[V], start[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = g.decay[ch + v];
    first[v] = g.saved[(static_cast<size_t>(seq) * g.n_saved + c * (T * W / kSavedEvery)) * g.D + ch + v];
    start[v] = g.glast != nullptr ? g.glast[static_cast<size_t>(seq) * g.D + ch + v] : 0.f;
  }
  Lane<E, V> x[T], in[T], r[T], z[T], gy[T];
#pragma unroll
  for (int k = 0; k < T; ++k) {
    const long long row = row0 + min(t0 + k, g.L - 1);
    r[k] = lane_load<E, V>(g.r + row * g.ld_r, ch);
    in[k] = lane_load<E, V>(g.i + row * g.ld_i, ch);
    x[k] = lane_load<E, V>(g.x + row * g.ld_x, ch);
    gy[k] = lane_load<E, V>(g.gy + row * g.ld_gy, ch);
    if (GATE) z[k] = lane_load<E, V>(g.z + row * g.ld_z, ch);
  }
  __builtin_amdgcn_sched_barrier(0);  // everything is asked for before anything is used
  float sum[V], h[V], M[V];
  // a, m g, g, sigmoid(r), a b / (1 - a^2), and what of gy reaches h and the output gate
  float a[T][V], mg[T][V], gate[T][V], open[T][V], back[T][V], go[T][V], gd[T][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = -decay_rate(rate[v], g.scale);
    sum[v] = h[v] = M[v] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < T; ++k) {
    const bool past = t0 + k >= g.L;  // l and go are zero there: nothing changes
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float rest;
      open[k][v] = sigmoid_of<kFull>(to_f(r[k].v[v]));
      gate[k][v] = sigmoid_of<kFull>(to_f(in[k].v[v]));
      const float l = past ? 0.f : rate[v] * open[k][v];
      decay_of<kFull>(l, a[k][v], rest);
      mg[k][v] = __builtin_amdgcn_sqrtf(rest) * gate[k][v];
      const float b = mg[k][v] * to_f(x[k].v[v]);
      back[k][v] = a[k][v] * b * __builtin_amdgcn_rcpf(rest + kTiny);  // where rest is zero, b is
      go[k][v] = past ? 0.f : to_f(gy[k].v[v]);
      if (GATE) {
        const float zz = to_f(z[k].v[v]), s = sigmoid_of<kFull>(zz);
        gd[k][v] = go[k][v] * (s * fmaf(zz, 1.f - s, 1.f));
        go[k][v] *= zz * s;
      }
      sum[v] += l;
      h[v] = fmaf(a[k][v], h[v], b);
    }
  }
  // what reaches the step before the wave's first, from a zero gradient behind its last
#pragma unroll
  for (int k = T - 1; k >= 0; --k)
#pragma unroll
    for (int v = 0; v < V; ++v) M[v] = a[k][v] * (go[k][v] + M[v]);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s_l[w][lane][v] = half_of(sum[v]);
    s_h[w][lane][v] = h[v];
  }
  const Rec rec{records, static_cast<size_t>(n_groups) * 64 * V};
  const size_t rec_ch = (static_cast<size_t>(group) * 64 + lane) * V;
  float carry[V];
  // the waves in the scan's order: the last first
  join_chunks<V, W, P>(s_join, W - 1 - w, lane, j, g.n_chunks, rec, rec_ch, sync, sum, M, start, carry);

  // the states again, from the chunk's start: the output gate's gradient, and what of them
  // the decay gate's needs
  float state[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    state[v] = first[v];
    for (int u = 0; u < w; ++u) state[v] = decayed(s_l[u][lane][v], state[v]) + s_h[u][lane][v];
  }
#pragma unroll
  for (int k = 0; k < T; ++k) {
    if (t0 + k >= g.L) break;
    Lane<E, V> oz;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      back[k][v] = state[v] - back[k][v];
      state[v] = fmaf(a[k][v], state[v], mg[k][v] * to_f(x[k].v[v]));
      if (GATE) oz.v[v] = from_f<E>(gd[k][v] * state[v]);
    }
    if (GATE && active) lane_store<E, V>(g.gz + (row0 + t0 + k) * g.ld_out, ch, oz);
  }
  float q_sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) q_sum[v] = 0.f;
#pragma unroll
  for (int k = T - 1; k >= 0; --k) {
    if (t0 + k >= g.L) continue;
    const long long at = (row0 + t0 + k) * g.ld_out;
    Lane<E, V> ox, oi, oR;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float G = go[k][v] + carry[v], gm = G * mg[k][v];
      ox.v[v] = from_f<E>(gm);
      oi.v[v] = from_f<E>(gm * to_f(x[k].v[v]) * (1.f - gate[k][v]));
      carry[v] = a[k][v] * G;
      const float q = carry[v] * (kLn2 * rate[v] * open[k][v]) * back[k][v];
      oR.v[v] = from_f<E>(q * (1.f - open[k][v]));
      q_sum[v] += q;
    }
    if (active) {
      lane_store<E, V>(g.gx + at, ch, ox);
      lane_store<E, V>(g.gi + at, ch, oi);
      lane_store<E, V>(g.gr + at, ch, oR);
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
// A channel or two a lane and no loop: the latency of three dependent loads (slot, state) is all there
// is, 3.4 us at [32, 2048]; every lane forms its own decay's rate.
template <class E, int V, bool GATE>
__global__ __launch_bounds__(256) void recurrence_step_kernel(Forward<E> g) {
  constexpr bool kFull = sizeof(E) == 4;
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int lanes = g.D / V;
  const long long row = at / lanes;
  if (row >= g.L) return;
  const unsigned ch = static_cast<unsigned>(at - row * lanes) * V;
  const int from = g.slots[row], to = g.out_slots[row];
  const bool have = from >= 0 && from < g.n_slots, keep = to >= 0 && to < g.n_slots;
  const Lane<E, V> r = lane_load<E, V>(g.r + row * g.ld_r, ch), in = lane_load<E, V>(g.i + row * g.ld_i, ch),
                   x = lane_load<E, V>(g.x + row * g.ld_x, ch);
  Lane<E, V> z{}, out;
  if (GATE) z = lane_load<E, V>(g.z + row * g.ld_z, ch);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float a, rest;
    decay_of<kFull>(-decay_rate(g.decay[ch + v], g.scale) * sigmoid_of<kFull>(to_f(r.v[v])), a, rest);
    float h = __builtin_amdgcn_sqrtf(rest) * (sigmoid_of<kFull>(to_f(in.v[v])) * to_f(x.v[v]));
    if (have) h = fmaf(a, g.pool[static_cast<size_t>(from) * g.D + ch + v], h);
    if (keep) g.pool[static_cast<size_t>(to) * g.D + ch + v] = h;
    if (GATE) {
      const float zz = to_f(z.v[v]);
      h *= zz * sigmoid_of<kFull>(zz);
    }
    out.v[v] = from_f<E>(have || keep ? h : 0.f);
  }
  lane_store<E, V>(g.y + row * g.D, ch, out);
}

// ---- launches -----------------------------------------------------------------------------
int64_t chunks_of(int64_t L, int steps) { return L > 0 ? (L + steps - 1) / steps : 1; }

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

// The records of a launch's chunks; one chunk a group hands nothing on and needs none, nor an
// order among its workgroups.
int records_of(StreamCall& call, int64_t total, int64_t n_chunks, int channels, void** records, LaunchSync* sync) {
  *records = nullptr;
  *sync = LaunchSync{};
  if (n_chunks == 1) return OSSM_OK;
  return acquire_scratch(call, static_cast<size_t>(total) * kRecords * channels * sizeof(unsigned long long), total, records, sync);
}

template <class E, int V, int T, int W, int P, bool PACKED>
int forward_tile(Forward<E> g, StreamCall& call) {
  g.n_cols = (g.D + 64 * V - 1) / (64 * V);
  g.n_chunks = static_cast<int>(chunks_of(g.L, T * W));
  const int64_t total = int64_t(g.B) * g.n_cols * g.n_chunks;
  if (int rc = check_grid(PACKED ? "recurrence_prompt" : "recurrence_forward", total, W * 64)) return rc;
  void* records = nullptr;
  LaunchSync sync{};
  if (int rc = records_of(call, total, g.n_chunks, 64 * V, &records, &sync)) return rc;
  const auto kern = g.z != nullptr ? recurrence_forward_kernel<E, V, T, W, P, PACKED, true>
                                   : recurrence_forward_kernel<E, V, T, W, P, PACKED, false>;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(total)), dim3(W * 64), 0, call.stream(), g,
                     static_cast<unsigned long long*>(records), sync);
  return launch_check("recurrence_forward_kernel");
}

// Steps a wave, waves and neighbours by how many groups of 64 V channels there are.  Few: the
// chunks' chain is what takes time, so chunks are long and many are joined at once.  Many: workgroups
// are small, so that some load while others compute or wait.  us, forward with a gate:
//   bf16, T W P    8 16 16   16 4 8   16 4 4  |  f32          8 16 16   16 8 16   16 4 4
//   16384 x 512       37.8              83.2  |  25600 x 128     24.7      27.9     93.6
//   16384 x 2048     111      108      114    |  8192 x 1024     43.0      44.6     58.3
//   65536 x 2048              344      385    |  2 x 8192 x 2048  155      136      151
//   2 x 8192 x 2048           101       99    |
//   4 x 8192 x 2048  208      166      163    |
template <class E, bool PACKED>
int forward(Forward<E> g, StreamCall& call) {
  if constexpr (sizeof(E) == 2) {
    const bool pairs = in_pairs<E>(g.D, {g.ld_x, g.ld_i, g.ld_r, g.z ? g.ld_z : 0}, {g.x, g.i, g.r, g.z, g.y});
    const int64_t groups = int64_t(g.B) * ((g.D + 127) / 128);
    if (pairs && groups >= 32) return forward_tile<E, 2, 16, 4, 4, PACKED>(g, call);
    if (pairs && groups >= 16) return forward_tile<E, 2, 16, 4, 8, PACKED>(g, call);
    if (pairs) return forward_tile<E, 2, 8, 16, 16, PACKED>(g, call);
  }
  return forward_tile<E, 1, 16, 8, 16, PACKED>(g, call);
}

template <class E, int V, int T, int W, int P>
int backward_tile(Backward<E> g, float* gdecay, StreamCall& call) {
  static_assert(T * W % kSavedEvery == 0, "a chunk starts at a saved state");
  g.n_cols = (g.D + 64 * V - 1) / (64 * V);
  g.n_chunks = static_cast<int>(chunks_of(g.L, T * W));
  const int64_t total = int64_t(g.B) * g.n_cols * g.n_chunks;
  if (int rc = check_grid("recurrence_backward", total, W * 64)) return rc;
  if (gdecay != nullptr) {
    void* p = nullptr;
    if (int rc = acquire_workspace(call, static_cast<size_t>(g.n_chunks) * g.B * g.D * sizeof(float), &p)) return rc;
    g.partial = static_cast<float*>(p);
  }
  void* records = nullptr;
  LaunchSync sync{};
  if (int rc = records_of(call, total, g.n_chunks, 64 * V, &records, &sync)) return rc;
  const auto kern = g.z != nullptr ? recurrence_backward_kernel<E, V, T, W, P, true> : recurrence_backward_kernel<E, V, T, W, P, false>;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(total)), dim3(W * 64), 0, call.stream(), g,
                     static_cast<unsigned long long*>(records), sync);
  if (int rc = launch_check("recurrence_backward_kernel")) return rc;
  if (gdecay == nullptr) return OSSM_OK;
  hipLaunchKernelGGL(decay_grad_kernel, dim3(static_cast<unsigned>((g.D + kSumColumns - 1) / kSumColumns)),
                     dim3(kSumThreads), 0, call.stream(), g.partial, g.n_chunks * g.B, g.D, g.decay, gdecay);
  return launch_check("decay_grad_kernel");
}

// As the forward's.  us: bf16, T W P   8 8 8   8 4 4  |  f32       8 16 16   8 8 8
//                    16384 x 512        58.3    128   |  25600 x 128    28.9    53.4
//                    16384 x 2048        184    186   |  8192 x 1024    69.2    67.1
//                    4 x 8192 x 2048     337    301   |  2 x 8192 x 2048  243    231
template <class E>
int backward(Backward<E> g, float* gdecay, StreamCall& call) {
  if constexpr (sizeof(E) == 2) {
    const bool pairs = in_pairs<E>(g.D, {g.ld_x, g.ld_i, g.ld_r, g.z ? g.ld_z : 0, g.ld_gy, g.ld_out},
                                   {g.x, g.i, g.r, g.z, g.gy, g.gx, g.gi, g.gr, g.gz});
    const int64_t groups = int64_t(g.B) * ((g.D + 127) / 128);
    if (pairs && groups >= 24) return backward_tile<E, 2, 8, 4, 4>(g, gdecay, call);
    if (pairs) return backward_tile<E, 2, 8, 8, 8>(g, gdecay, call);
  }
  return backward_tile<E, 1, 8, 16, 16>(g, gdecay, call);
}

int check_sizes(const char* what, int dtype, float scale, int64_t B, int64_t L, int64_t D) {
  if (dtype != OSSM_F32 && dtype != OSSM_BF16)
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": unknown dtype");
  // the root of 1 - a^2 is none where a passes one
  if (!(scale > 0.f && scale < __builtin_inff()))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": scale must be positive and finite");
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
  return batch * chunks_of(length, kSavedEvery) * dim;
}

int ossm_recurrence_forward(int dtype, const void* x, int64_t ld_x, const void* input_gate, int64_t ld_input_gate,
                            const void* decay_gate, int64_t ld_decay_gate, const void* output_gate, int64_t ld_output_gate,
                            const float* decay, float scale, const float* start, void* y, float* last, float* saved,
                            int64_t batch, int64_t length, int64_t dim, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "recurrence_forward";
  if (int rc = check_sizes(what, dtype, scale, batch, length, dim)) return rc;
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
    g.n_saved = static_cast<int>(chunks_of(length, kSavedEvery));
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
  if (int rc = check_sizes(what, dtype, scale, batch, length, dim)) return rc;
  if (batch == 0 || length == 0 || dim == 0) return OSSM_OK;
  if (!grad_y || !x || !input_gate || !decay_gate || !decay || !saved || !grad_x || !grad_input_gate || !grad_decay_gate ||
      (output_gate != nullptr) != (grad_output_gate != nullptr))
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
    g.n_saved = static_cast<int>(chunks_of(length, kSavedEvery));
    return backward(g, grad_decay, call);
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
  if (int rc = check_sizes(what, dtype, scale, n_seqs, rows, dim)) return rc;
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
    if (rows == 0) {  // the kernel loads before it looks at the length: from a row that is there
      g.x = g.i = g.r = reinterpret_cast<const E*>(decay);
      if (g.z != nullptr) g.z = g.x;
    }
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
  if (int rc = check_sizes(what, dtype, scale, 1, rows, dim)) return rc;
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
        hipLaunchKernelGGL((g.z ? recurrence_step_kernel<E, 2, true> : recurrence_step_kernel<E, 2, false>),
                           dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, g);
        return launch_check("recurrence_step_kernel");
      }
    hipLaunchKernelGGL((g.z ? recurrence_step_kernel<E, 1, true> : recurrence_step_kernel<E, 1, false>),
                       dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, g);
    return launch_check("recurrence_step_kernel");
  };
  return dtype == OSSM_BF16 ? go(bf16_t{}) : go(0.f);
}

}  // extern "C"
