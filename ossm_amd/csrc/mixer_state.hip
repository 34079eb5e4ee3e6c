// The Mamba mixer between its in and out projections, with states kept in a pool:
// packed ragged prompts (ossm_mixer_prompt) and single tokens (ossm_mixer_step).
//
//   u_t  = silu(cb + sum_k cw[k] x[t - K + 1 + k])        x, z the halves of xz
//   p_t  = Wx u_t,   dt_t = softplus(Wdt p_t[:R] + bias)   B, C the rest of p_t
//   h_t  = exp(dt_t A) h_{t-1} + dt_t u_t B_t,  A = -exp(A_log)
//   y_t  = (C_t . h_t + skip u_t) silu(z_t)
//
// All of it in float32 whatever E is: u, p, dt and h are never rounded to E (h is an
// output in float32, and a u rounded to bf16 would leave 2^-9 in it).
//
// A token's launches: mixer_proj_kernel (conv, its state's update, x_proj over a block
// of channels) and mixer_token_kernel (the blocks' sums, dt, the state's update, the
// gate).  x_proj sums over all channels, so two launches is the least.
//
// A prompt batch is one row of packed tokens cut into chunks of equal length,
// whatever the prompts' lengths (the host never reads the offsets): a prompt's
// first token resets the recurrence, so a chunk may hold many prompts or a
// piece of one.  mixer_scan_kernel<summary> finds what each chunk leaves to a zero
// carry and the sum of its dt (the decay over the chunk is exp(A sum dt)),
// mixer_carry_kernel folds the chunks in order, mixer_scan_kernel<output> walks the
// chunks again from their carries.  One chunk needs the last only.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>

#include "../../include/ossm_lm.h"
#include "lm_types.hpp"
#include "runtime.hpp"
#include "scan_device.hpp"

namespace ossm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxConv = 8;
constexpr int kProjThreads = 256;
constexpr int kProjWaves = kProjThreads / kWave;
constexpr int kSub = 32;                       // channels of one wave's share of x_proj
constexpr int kProjBlock = kProjWaves * kSub;  // channels of a workgroup

template <class E>
struct Mixer {
  const E* xz;
  const E* conv_w;
  const E* conv_b;
  const E* x_proj;
  const E* dt_proj;
  const float* dt_bias;
  const float* a_log;
  const float* skip;
  E* conv_state;
  float* ssm;
  const int32_t* in_slots;
  const int32_t* out_slots;
  const int32_t* offsets;  // null for single tokens
  const uint8_t* resume;
  E* y;
  float* part;   // [n_blocks][rows][Nc]: x_proj's sums over blocks of channels
  float* u;      // tokens: [rows][Di]
  float* bc;     // prompts: [rows][2][Npad], B and C, zero from N on
  float* dt;     // prompts: [rows][Di]
  float* local;  // prompts: [n_chunks][N][Di], a chunk's end from a zero carry
  float* carry;  // prompts: [n_chunks][N][Di], the state before a chunk
  float* sum_dt; // prompts: [n_chunks][Di], negative where a prompt starts in the chunk
  float* init;   // prompts: [n_seqs][N][Di] copies of the resumed states, or null
  float* y_sum;  // prompts with N past a block of states: [rows][Di]
  long long ld;
  int rows, n_seqs, n_slots, Di, N, R, K, Nc, Npad, n_blocks, chunk, n_chunks;
};

// Where sequence i starts, in range whatever the offsets hold.
template <class E>
__device__ __forceinline__ int offset_of(const Mixer<E>& g, int i) { return min(max(g.offsets[i], 0), g.rows); }

// The last sequence that starts at or before token t (-1: none).
template <class E>
__device__ __forceinline__ int seq_of(const Mixer<E>& g, int t) {
  int lo = 0, hi = g.n_seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (offset_of(g, mid) <= t) lo = mid + 1; else hi = mid;
  }
  return lo - 1;
}

template <class E>
__device__ __forceinline__ bool in_pool(const Mixer<E>& g, int slot) { return slot >= 0 && slot < g.n_slots; }

// The slot that sequence s continues from, -1 where it starts from zeros.
template <class E>
__device__ __forceinline__ int start_slot(const Mixer<E>& g, int s) {
  if (g.offsets != nullptr && (g.resume == nullptr || g.resume[s] == 0)) return -1;
  const int slot = g.in_slots[s];
  return in_pool(g, slot) ? slot : -1;
}

// The conv's input at position pos of a sequence that starts at row `start` (pos < start:
// from the slot's last inputs).
template <class E>
__device__ __forceinline__ float conv_input(const Mixer<E>& g, int pos, int start, int slot, int d) {
  if (pos >= start) return to_f(g.xz[static_cast<size_t>(pos) * g.ld + d]);
  const int j = g.K - 1 + pos - start;
  if (slot < 0 || j < 0) return 0.f;
  return to_f(g.conv_state[(static_cast<size_t>(slot) * (g.K - 1) + j) * g.Di + d]);
}

// Eight consecutive weights (zeros past the row's n), vector loads where `vec`.
__device__ __forceinline__ void load8(const float* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}
__device__ __forceinline__ void load8(const bf16_t* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f(p[i]) : 0.f;
  }
}

// conv + SiLU of RB rows over a block of channels, and x_proj's partial sums over it.
// Each wave takes kSub of the channels and all Nc outputs, 64 at a time, one per lane;
// the waves' sums meet in LDS in a fixed order.
template <class E, int RB, bool PROMPT>
__global__ __launch_bounds__(kProjThreads) void mixer_proj_kernel(Mixer<E> g, bool vec) {
  __shared__ float s_u[RB][kProjBlock];
  __shared__ float s_sum[kProjWaves][RB][kWave];
  __shared__ int s_start[RB], s_slot[RB];
  const int blk = static_cast<int>(blockIdx.x % g.n_blocks);
  const int r0 = static_cast<int>(blockIdx.x / g.n_blocks) * RB;
  const int c0 = blk * kProjBlock;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = wave_id();
  if (tid < RB) {
    const int r = r0 + tid;
    int start = INT_MAX, slot = -1;  // INT_MAX: padding
    if (r < g.rows) {
      if constexpr (PROMPT) {
        const int s = seq_of(g, r);
        if (s >= 0 && r < offset_of(g, s + 1)) { start = offset_of(g, s); slot = start_slot(g, s); }
      } else {
        start = r;
        slot = start_slot(g, r);
      }
    }
    s_start[tid] = start;
    s_slot[tid] = slot;
  }
  __syncthreads();
  for (int i = tid; i < RB * kProjBlock; i += kProjThreads) {
    const int rr = i / kProjBlock, c = i % kProjBlock, r = r0 + rr, d = c0 + c;
    float u = 0.f;
    if (d < g.Di && s_start[rr] != INT_MAX) {
      float p = g.conv_b != nullptr ? to_f(g.conv_b[d]) : 0.f;
      if constexpr (PROMPT) {
        for (int k = 0; k < g.K; ++k)
          p = fmaf(to_f(g.conv_w[static_cast<size_t>(d) * g.K + k]),
                   conv_input(g, r - g.K + 1 + k, s_start[rr], s_slot[rr], d), p);
        u = silu_f(p);
      } else {
        float x[kMaxConv];
#pragma unroll
        for (int k = 0; k < kMaxConv; ++k)
          if (k < g.K) {
            x[k] = conv_input(g, r - g.K + 1 + k, r, s_slot[rr], d);
            p = fmaf(to_f(g.conv_w[static_cast<size_t>(d) * g.K + k]), x[k], p);
          }
        u = silu_f(p);
        const int out = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[r];
        if (in_pool(g, out)) {
#pragma unroll
          for (int k = 1; k < kMaxConv; ++k)
            if (k < g.K)
              g.conv_state[(static_cast<size_t>(out) * (g.K - 1) + k - 1) * g.Di + d] = from_f<E>(x[k]);
        }
        g.u[static_cast<size_t>(r) * g.Di + d] = u;
      }
    }
    s_u[rr][c] = u;
  }
  __syncthreads();
  for (int j0 = 0; j0 < g.Nc; j0 += kWave) {
    const int j = min(j0 + lane, g.Nc - 1);
    float acc[RB];
#pragma unroll
    for (int rr = 0; rr < RB; ++rr) acc[rr] = 0.f;
#pragma unroll
    for (int q = 0; q < kSub; q += 8) {
      const int c = w * kSub + q;
      float wt[8];
      const int left = g.Di - (c0 + c);
      load8(g.x_proj + static_cast<size_t>(j) * g.Di + (left > 0 ? c0 + c : 0), left, vec, wt);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int rr = 0; rr < RB; ++rr) acc[rr] = fmaf(wt[i], s_u[rr][c + i], acc[rr]);
    }
#pragma unroll
    for (int rr = 0; rr < RB; ++rr) s_sum[w][rr][lane] = acc[rr];
    __syncthreads();
    for (int i = tid; i < RB * kWave; i += kProjThreads) {
      const int rr = i / kWave, l = i % kWave;
      if (r0 + rr < g.rows && j0 + l < g.Nc) {
        float s = s_sum[0][rr][l];
#pragma unroll
        for (int v = 1; v < kProjWaves; ++v) s += s_sum[v][rr][l];
        g.part[(static_cast<size_t>(blk) * g.rows + r0 + rr) * g.Nc + j0 + l] = s;
      }
    }
    __syncthreads();
  }
}

// s_p[RB][Nc] = the rows' projections, from the blocks' partial sums.
template <int RB, class E>
__device__ __forceinline__ void sum_proj(const Mixer<E>& g, int r0, float* s_p) {
  const size_t step = static_cast<size_t>(g.rows) * g.Nc;
  for (int i = threadIdx.x; i < RB * g.Nc; i += blockDim.x) {
    const int r = r0 + i / g.Nc;
    float s = 0.f;
    if (r < g.rows) {
      const float* p = g.part + static_cast<size_t>(r) * g.Nc + i % g.Nc;
#pragma unroll 8
      for (int b = 0; b < g.n_blocks; ++b) s += p[b * step];
    }
    s_p[i] = s;
  }
}

// dt of RB rows at channel d from their projections in LDS.
template <int RB, class E>
__device__ __forceinline__ void dt_of(const Mixer<E>& g, const float* s_p, int d, bool vec, float (&dt)[RB]) {
  const float bias = g.dt_bias[d];
#pragma unroll
  for (int rr = 0; rr < RB; ++rr) dt[rr] = bias;
  for (int q = 0; q < g.R; q += 8) {
    float wt[8];
    load8(g.dt_proj + static_cast<size_t>(d) * g.R + q, g.R - q, vec, wt);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = min(q + i, g.Nc - 1);  // past R the weight is zero; what it meets is finite or replaced
#pragma unroll
      for (int rr = 0; rr < RB; ++rr) {
        const float p = s_p[rr * g.Nc + k];
        dt[rr] = q + i < g.R ? fmaf(wt[i], p, dt[rr]) : dt[rr];
      }
    }
  }
#pragma unroll
  for (int rr = 0; rr < RB; ++rr) dt[rr] = softplus_f(dt[rr]);
}

// One token: a thread per channel, RB rows one after another.
template <class E, int RB>
__global__ __launch_bounds__(256) void mixer_token_kernel(Mixer<E> g, bool vec) {
  extern __shared__ float s_p[];  // [RB][Nc]
  const int r0 = static_cast<int>(blockIdx.y) * RB;
  sum_proj<RB>(g, r0, s_p);
  __syncthreads();
  const int d = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x);
  if (d >= g.Di) return;
  float dt[RB];
  dt_of<RB>(g, s_p, d, vec, dt);
  const float skip = g.skip != nullptr ? g.skip[d] : 0.f;
#pragma unroll
  for (int rr = 0; rr < RB; ++rr) {
    const int r = r0 + rr;
    if (r >= g.rows) break;
    const int in = start_slot(g, r);
    const int to = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[r];
    const bool keep = in_pool(g, to);
    E* out = g.y + static_cast<size_t>(r) * g.Di + d;
    if (in < 0 && !keep) { *out = from_f<E>(0.f); continue; }
    const float u = g.u[static_cast<size_t>(r) * g.Di + d];
    const float z = to_f(g.xz[static_cast<size_t>(r) * g.ld + g.Di + d]);
    const float* B = s_p + rr * g.Nc + g.R;
    const float* C = B + g.N;
    const float* hi = g.ssm + (static_cast<size_t>(in < 0 ? 0 : in) * g.N) * g.Di + d;
    float* ho = g.ssm + (static_cast<size_t>(keep ? to : 0) * g.N) * g.Di + d;
    const float du = dt[rr] * u;
    float y = skip * u;
    for (int n0 = 0; n0 < g.N; n0 += 16) {
      float h[16], a[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int n = min(n0 + i, g.N - 1);
        h[i] = in >= 0 ? hi[static_cast<size_t>(n) * g.Di] : 0.f;
        a[i] = g.a_log[static_cast<size_t>(d) * g.N + n];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (n0 + i >= g.N) break;
        const float decay = __builtin_amdgcn_exp2f(-expf(a[i]) * kLog2e * dt[rr]);
        const float v = fmaf(decay, h[i], du * B[n0 + i]);
        y = fmaf(C[n0 + i], v, y);
        if (keep) ho[static_cast<size_t>(n0 + i) * g.Di] = v;
      }
    }
    *out = from_f<E>(y * silu_f(z));
  }
}

// Prompts: B, C and dt of every token, from x_proj's partial sums.
template <class E, int RB>
__global__ __launch_bounds__(256) void mixer_dt_kernel(Mixer<E> g, bool vec) {
  extern __shared__ float s_p[];  // [RB][Nc]
  const int nb = (g.Di + 255) / 256;
  const int r0 = static_cast<int>(blockIdx.x / nb) * RB, cb = static_cast<int>(blockIdx.x % nb);
  sum_proj<RB>(g, r0, s_p);
  __syncthreads();
  if (cb == 0) {
    for (int i = threadIdx.x; i < RB * 2 * g.Npad; i += blockDim.x) {
      const int rr = i / (2 * g.Npad), k = i % (2 * g.Npad), half = k / g.Npad, n = k % g.Npad;
      if (r0 + rr < g.rows)
        g.bc[static_cast<size_t>(r0 + rr) * 2 * g.Npad + k] =
            n < g.N ? s_p[rr * g.Nc + g.R + half * g.N + n] : 0.f;
    }
  }
  const int d = cb * 256 + static_cast<int>(threadIdx.x);
  if (d >= g.Di) return;
  float dt[RB];
  dt_of<RB>(g, s_p, d, vec, dt);
#pragma unroll
  for (int rr = 0; rr < RB; ++rr)
    if (r0 + rr < g.rows) g.dt[static_cast<size_t>(r0 + rr) * g.Di + d] = dt[rr];
}

// The resumed states, copied before the scan that may overwrite their slots.
template <class E>
__global__ __launch_bounds__(256) void mixer_gather_kernel(Mixer<E> g) {
  const int s = static_cast<int>(blockIdx.y);
  const int slot = start_slot(g, s);
  if (slot < 0) return;
  const size_t n = static_cast<size_t>(g.N) * g.Di;
  for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<size_t>(gridDim.x) * 256)
    g.init[s * n + i] = g.ssm[slot * n + i];
}

constexpr int kScanThreads = 128;
constexpr int kGroup = 4;  // tokens whose inputs are loaded together

// One thread per channel walks a chunk.  NB states in registers (from n_base), KT conv
// taps (taps before the last K are skipped).  OUT: from the chunk's carry, writing y and
// the states of the prompts that end here; else from the last prompt start in the chunk
// (or a zero carry), leaving the chunk's end and its sum of dt.
template <class E, int NB, int KT, bool OUT>
__global__ __launch_bounds__(kScanThreads) void mixer_scan_kernel(Mixer<E> g, const float* __restrict__ bc, int n_base) {
  const int d = static_cast<int>(blockIdx.x) * kScanThreads + static_cast<int>(threadIdx.x);
  if (d >= g.Di) return;
  const int c = static_cast<int>(blockIdx.y);
  const int t0 = c * g.chunk, t1 = min(t0 + g.chunk, g.rows);
  const bool last_block = n_base + NB >= g.N;
  float a2[NB], h[NB], cw[KT], win[KT - 1];
#pragma unroll
  for (int i = 0; i < NB; ++i)
    a2[i] = n_base + i < g.N ? -expf(g.a_log[static_cast<size_t>(d) * g.N + n_base + i]) * kLog2e : 0.f;
  const int skip_taps = KT - g.K;
#pragma unroll
  for (int k = 0; k < KT; ++k) cw[k] = k >= skip_taps ? to_f(g.conv_w[static_cast<size_t>(d) * g.K + k - skip_taps]) : 0.f;
#pragma unroll
  for (int i = 0; i < NB; ++i) h[i] = 0.f;
  const float cb = g.conv_b != nullptr ? to_f(g.conv_b[d]) : 0.f;
  const float skip = g.skip != nullptr ? g.skip[d] : 0.f;

  int s = seq_of(g, OUT ? t0 : t1 - 1);
  int t = t0;
  float dt_sum = 0.f;
  if constexpr (!OUT) {
    if (s < 0) return;  // padding only: the next chunk starts a prompt
    const int start = offset_of(g, s);
    if (start >= t0) { t = start; dt_sum = -1.f; }
  }
  while (t < t1) {
    // the segment [t, e) of sequence s
    int e, start = 0, slot = -1;
    bool inside = false;
    if (s >= 0 && t < offset_of(g, s + 1)) {
      inside = true;
      start = offset_of(g, s);
      e = min(t1, offset_of(g, s + 1));
      slot = start_slot(g, s);
    } else {
      e = s + 1 < g.n_seqs ? min(t1, max(offset_of(g, s + 1), t + 1)) : t1;  // padding
    }
    if (!inside) {
      if constexpr (OUT)
        if (last_block)
          for (int i = t; i < e; ++i) g.y[static_cast<size_t>(i) * g.Di + d] = from_f<E>(0.f);
      t = e;
    } else {
      if (t == start) {
        const float* src = g.init != nullptr ? g.init + (static_cast<size_t>(s) * g.N) * g.Di
                                             : g.ssm + (static_cast<size_t>(max(slot, 0)) * g.N) * g.Di;
#pragma unroll
        for (int i = 0; i < NB; ++i)
          h[i] = slot >= 0 && n_base + i < g.N ? src[static_cast<size_t>(n_base + i) * g.Di + d] : 0.f;
      } else {
        const bool carried = OUT && t == t0 && c > 0;
        const float* src = g.carry + (static_cast<size_t>(c) * g.N) * g.Di;
#pragma unroll
        for (int i = 0; i < NB; ++i)
          h[i] = carried && n_base + i < g.N ? src[static_cast<size_t>(n_base + i) * g.Di + d] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < KT - 1; ++k) {
        const int pos = t - (KT - 1) + k;
        win[k] = k >= skip_taps ? conv_input(g, pos, start, slot, d) : 0.f;
      }
      for (; t < e; t += kGroup) {
        float x[kGroup], z[kGroup], dt[kGroup], ys[kGroup];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const size_t r = static_cast<size_t>(min(t + i, e - 1));
          x[i] = to_f(g.xz[r * g.ld + d]);
          dt[i] = g.dt[r * g.Di + d];
          if constexpr (OUT) {
            z[i] = to_f(g.xz[r * g.ld + g.Di + d]);
            ys[i] = n_base > 0 ? g.y_sum[r * g.Di + d] : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          if (t + i >= e) break;
          const float* B = bc + static_cast<size_t>(t + i) * 2 * g.Npad + n_base;
          const float* C = B + g.Npad;
          float p = cb;
#pragma unroll
          for (int k = 0; k < KT - 1; ++k)
            if (k >= skip_taps) p = fmaf(cw[k], win[k], p);
          p = fmaf(cw[KT - 1], x[i], p);
#pragma unroll
          for (int k = 0; k + 1 < KT - 1; ++k) win[k] = win[k + 1];
          if constexpr (KT > 1) win[KT - 2] = x[i];
          const float u = silu_f(p);
          const float du = dt[i] * u;
          float y = OUT && n_base == 0 ? skip * u : ys[i];
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const float decay = __builtin_amdgcn_exp2f(a2[n] * dt[i]);
            h[n] = fmaf(decay, h[n], du * B[n]);
            if constexpr (OUT) y = fmaf(C[n], h[n], y);
          }
          if constexpr (OUT) {
            const size_t at = static_cast<size_t>(t + i) * g.Di + d;
            if (last_block) g.y[at] = from_f<E>(y * silu_f(z[i]));
            else g.y_sum[at] = y;
          } else if (dt_sum >= 0.f) {
            dt_sum += dt[i];
          }
        }
      }
      t = e;
      if constexpr (OUT) {
        if (e == offset_of(g, s + 1)) {
          const int to = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[s];
          if (in_pool(g, to)) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
              if (n_base + i < g.N)
                g.ssm[(static_cast<size_t>(to) * g.N + n_base + i) * g.Di + d] = h[i];
          }
        }
      }
    }
    // the sequence at t (empty ones are passed by; their states are the finish kernel's)
    while (s + 1 < g.n_seqs && offset_of(g, s + 1) <= t) ++s;
  }
  if constexpr (!OUT) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (n_base + i < g.N) g.local[(static_cast<size_t>(c) * g.N + n_base + i) * g.Di + d] = h[i];
    if (n_base == 0) g.sum_dt[static_cast<size_t>(c) * g.Di + d] = dt_sum;
  }
}

// carry[c + 1] = exp(A sum_dt[c]) carry[c] + local[c], a thread per state.
template <class E>
__global__ __launch_bounds__(256) void mixer_carry_kernel(Mixer<E> g) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const size_t nd = static_cast<size_t>(g.N) * g.Di;
  if (i >= nd) return;
  const int n = static_cast<int>(i / g.Di), d = static_cast<int>(i % g.Di);
  const float a2 = -expf(g.a_log[static_cast<size_t>(d) * g.N + n]) * kLog2e;
  float h = 0.f;
  constexpr int kAhead = 8;
  for (int c0 = 0; c0 + 1 < g.n_chunks; c0 += kAhead) {
    float l[kAhead], sd[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = min(c0 + k, g.n_chunks - 2);
      l[k] = g.local[c * nd + i];
      sd[k] = g.sum_dt[static_cast<size_t>(c) * g.Di + d];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (c0 + k + 1 >= g.n_chunks) break;
      h = sd[k] < 0.f ? l[k] : fmaf(__builtin_amdgcn_exp2f(a2 * sd[k]), h, l[k]);
      g.carry[(c0 + k + 1) * nd + i] = h;
    }
  }
}

// Every prompt's last K - 1 inputs, and the states of empty prompts.
template <class E>
__global__ __launch_bounds__(256) void mixer_finish_kernel(Mixer<E> g) {
  const int d = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
  if (d >= g.Di) return;
  const int s = static_cast<int>(blockIdx.y);
  const int to = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[s];
  if (!in_pool(g, to)) return;
  const int start = offset_of(g, s), end = max(offset_of(g, s + 1), start);
  const int slot = start_slot(g, s);
  float x[kMaxConv - 1];
#pragma unroll
  for (int k = 0; k < kMaxConv - 1; ++k)
    if (k < g.K - 1) x[k] = conv_input(g, end - (g.K - 1) + k, start, slot, d);
#pragma unroll
  for (int k = 0; k < kMaxConv - 1; ++k)
    if (k < g.K - 1) g.conv_state[(static_cast<size_t>(to) * (g.K - 1) + k) * g.Di + d] = from_f<E>(x[k]);
  if (start == end && to != slot)
    for (int n = 0; n < g.N; ++n)
      g.ssm[(static_cast<size_t>(to) * g.N + n) * g.Di + d] =
          slot >= 0 ? g.ssm[(static_cast<size_t>(slot) * g.N + n) * g.Di + d] : 0.f;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class E, int NB, int KT>
int launch_scan(const Mixer<E>& g, bool out, int n_base, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((g.Di + kScanThreads - 1) / kScanThreads), static_cast<unsigned>(g.n_chunks));
  if (out)
    hipLaunchKernelGGL((mixer_scan_kernel<E, NB, KT, true>), grid, dim3(kScanThreads), 0, st, g, g.bc, n_base);
  else
    hipLaunchKernelGGL((mixer_scan_kernel<E, NB, KT, false>), grid, dim3(kScanThreads), 0, st, g, g.bc, n_base);
  return launch_check("mixer_scan_kernel");
}

template <class E>
int launch_scans(const Mixer<E>& g, bool out, hipStream_t st) {
  for (int n_base = 0; n_base < g.N; n_base += 32) {
    const int left = g.N - n_base;
    const bool k4 = g.K <= 4;
    int rc;
    if (left <= 8) rc = k4 ? launch_scan<E, 8, 4>(g, out, n_base, st) : launch_scan<E, 8, 8>(g, out, n_base, st);
    else if (left <= 16) rc = k4 ? launch_scan<E, 16, 4>(g, out, n_base, st) : launch_scan<E, 16, 8>(g, out, n_base, st);
    else rc = k4 ? launch_scan<E, 32, 4>(g, out, n_base, st) : launch_scan<E, 32, 8>(g, out, n_base, st);
    if (rc) return rc;
  }
  return OSSM_OK;
}

template <class E>
bool vec8(const E* p, int row) { return aligned16(p) && row % (16 / static_cast<int>(sizeof(E))) == 0; }

template <class E>
int step(Mixer<E> g, StreamCall& call, hipStream_t st) {
  g.n_blocks = (g.Di + kProjBlock - 1) / kProjBlock;
  const size_t part = static_cast<size_t>(g.n_blocks) * g.rows * g.Nc;
  void* ws = nullptr;
  if (int rc = acquire_workspace(call, (part + static_cast<size_t>(g.rows) * g.Di) * sizeof(float), &ws)) return rc;
  g.part = static_cast<float*>(ws);
  g.u = g.part + part;
  const bool vx = vec8(g.x_proj, g.Di), vd = vec8(g.dt_proj, g.R);
  const bool many = g.rows >= 32;
  const int rb = many ? 8 : 1;
  const dim3 ga(static_cast<unsigned>(g.n_blocks * ((g.rows + rb - 1) / rb)));
  if (many) hipLaunchKernelGGL((mixer_proj_kernel<E, 8, false>), ga, dim3(kProjThreads), 0, st, g, vx);
  else hipLaunchKernelGGL((mixer_proj_kernel<E, 1, false>), ga, dim3(kProjThreads), 0, st, g, vx);
  if (int rc = launch_check("mixer_proj_kernel")) return rc;
  const int rt = many ? 4 : 1, threads = many ? 256 : 64;
  const dim3 gb(static_cast<unsigned>((g.Di + threads - 1) / threads), static_cast<unsigned>((g.rows + rt - 1) / rt));
  const size_t lds = static_cast<size_t>(rt) * g.Nc * sizeof(float);
  if (many) hipLaunchKernelGGL((mixer_token_kernel<E, 4>), gb, dim3(threads), lds, st, g, vd);
  else hipLaunchKernelGGL((mixer_token_kernel<E, 1>), gb, dim3(threads), lds, st, g, vd);
  return launch_check("mixer_token_kernel");
}

template <class E>
int prompt(Mixer<E> g, StreamCall& call, hipStream_t st) {
  g.n_blocks = (g.Di + kProjBlock - 1) / kProjBlock;
  g.Npad = g.N <= 8 ? 8 : g.N <= 16 ? 16 : (g.N + 31) / 32 * 32;
  // enough chunks for four waves on each SIMD, of 16 tokens at least
  const int64_t waves = (g.Di + kWave - 1) / kWave;
  const int64_t want = std::max<int64_t>(1, 16 * std::max(1, device_cu_count(call.device())) / waves);
  g.chunk = static_cast<int>(std::max<int64_t>({16, (g.rows + want - 1) / want, (g.rows + 65534) / 65535}));
  g.n_chunks = (g.rows + g.chunk - 1) / g.chunk;
  const size_t nd = static_cast<size_t>(g.N) * g.Di;
  const bool carries = g.n_chunks > 1;
  size_t at = 0;
  const auto take = [&](size_t n) { const size_t o = at; at += (n + 63) / 64 * 64; return o; };
  const size_t o_part = take(static_cast<size_t>(g.n_blocks) * g.rows * g.Nc);
  const size_t o_bc = take(static_cast<size_t>(g.rows) * 2 * g.Npad);
  const size_t o_dt = take(static_cast<size_t>(g.rows) * g.Di);
  const size_t o_local = take(carries ? g.n_chunks * nd : 0);
  const size_t o_carry = take(carries ? g.n_chunks * nd : 0);
  const size_t o_sum = take(carries ? static_cast<size_t>(g.n_chunks) * g.Di : 0);
  const size_t o_init = take(g.resume != nullptr ? g.n_seqs * nd : 0);
  const size_t o_y = take(g.N > 32 ? static_cast<size_t>(g.rows) * g.Di : 0);
  void* ws = nullptr;
  if (int rc = acquire_workspace(call, at * sizeof(float), &ws)) return rc;
  float* f = static_cast<float*>(ws);
  g.part = f + o_part;
  g.bc = f + o_bc;
  g.dt = f + o_dt;
  g.local = f + o_local;
  g.carry = f + o_carry;
  g.sum_dt = f + o_sum;
  g.y_sum = f + o_y;
  if (g.rows > 0) {
    constexpr int RB = 8;
    const int64_t groups = (g.rows + RB - 1) / RB;
    hipLaunchKernelGGL((mixer_proj_kernel<E, RB, true>), dim3(static_cast<unsigned>(groups * g.n_blocks)),
                       dim3(kProjThreads), 0, st, g, vec8(g.x_proj, g.Di));
    if (int rc = launch_check("mixer_proj_kernel")) return rc;
    hipLaunchKernelGGL((mixer_dt_kernel<E, RB>), dim3(static_cast<unsigned>(groups * ((g.Di + 255) / 256))), dim3(256),
                       static_cast<size_t>(RB) * g.Nc * sizeof(float), st, g, vec8(g.dt_proj, g.R));
    if (int rc = launch_check("mixer_dt_kernel")) return rc;
    if (g.resume != nullptr) {
      g.init = f + o_init;
      hipLaunchKernelGGL(mixer_gather_kernel<E>, dim3(static_cast<unsigned>(std::min<size_t>(64, (nd + 255) / 256)),
                                                      static_cast<unsigned>(g.n_seqs)), dim3(256), 0, st, g);
      if (int rc = launch_check("mixer_gather_kernel")) return rc;
    }
    if (carries) {
      if (int rc = launch_scans(g, false, st)) return rc;
      hipLaunchKernelGGL(mixer_carry_kernel<E>, dim3(static_cast<unsigned>((nd + 255) / 256)), dim3(256), 0, st, g);
      if (int rc = launch_check("mixer_carry_kernel")) return rc;
    }
    if (int rc = launch_scans(g, true, st)) return rc;
  }
  hipLaunchKernelGGL(mixer_finish_kernel<E>, dim3(static_cast<unsigned>((g.Di + 255) / 256), static_cast<unsigned>(g.n_seqs)),
                     dim3(256), 0, st, g);
  return launch_check("mixer_finish_kernel");
}

int check_mixer(const char* what, int dtype, int64_t rows, int64_t n_seqs, int64_t n_slots, int64_t di, int64_t n,
                int64_t r, int64_t k, int64_t ld) {
  const std::string w(what);
  if (dtype != OSSM_F32 && dtype != OSSM_BF16) return set_error(OSSM_ERR_INVALID_ARGUMENT, w + ": unknown dtype");
  if (rows < 0 || n_seqs < 0 || n_slots < 0 || di < 0 || n < 1 || r < 1)
    return set_error(OSSM_ERR_INVALID_ARGUMENT, w + ": bad size");
  if (k < 1 || k > kMaxConv)
    return set_error(OSSM_ERR_UNSUPPORTED, w + ": conv widths 1.." + std::to_string(kMaxConv) + " supported, got " +
                                               std::to_string(k));
  if (rows > 1 && ld < 2 * di) return set_error(OSSM_ERR_INVALID_ARGUMENT, w + ": row stride of xz below 2 d_inner");
  if (rows > (1 << 24) || n_seqs > 65535 || n_slots > INT_MAX / 8 || di > (1 << 20) || n > 1024 || r + 2 * n > 2048 ||
      ((rows + 7) / 8) * ((di + 127) / 128) > INT_MAX / 2)
    return set_error(OSSM_ERR_UNSUPPORTED, w + ": size exceeds launch limits");
  return OSSM_OK;
}

template <class E>
Mixer<E> make(const void* xz, int64_t ld, const void* cw, const void* cb, const void* xp, const void* dp,
              const float* dtb, const float* al, const float* skip, void* cs, float* ssm, const int32_t* in,
              const int32_t* out, const int32_t* offs, const uint8_t* res, void* y, int64_t rows, int64_t n_seqs,
              int64_t n_slots, int64_t di, int64_t n, int64_t r, int64_t k) {
  Mixer<E> g{};
  g.xz = static_cast<const E*>(xz);
  g.conv_w = static_cast<const E*>(cw);
  g.conv_b = static_cast<const E*>(cb);
  g.x_proj = static_cast<const E*>(xp);
  g.dt_proj = static_cast<const E*>(dp);
  g.dt_bias = dtb;
  g.a_log = al;
  g.skip = skip;
  g.conv_state = static_cast<E*>(cs);
  g.ssm = ssm;
  g.in_slots = in;
  g.out_slots = out;
  g.offsets = offs;
  g.resume = res;
  g.y = static_cast<E*>(y);
  g.ld = ld;
  g.rows = static_cast<int>(rows);
  g.n_seqs = static_cast<int>(n_seqs);
  g.n_slots = static_cast<int>(n_slots);
  g.Di = static_cast<int>(di);
  g.N = static_cast<int>(n);
  g.R = static_cast<int>(r);
  g.K = static_cast<int>(k);
  g.Nc = g.R + 2 * g.N;
  return g;
}

}  // namespace
}  // namespace ossm

using namespace ossm;

extern "C" {

int ossm_lm_abi_version(void) { return 1; }

int ossm_mixer_step(int dtype, const void* xz, int64_t ld_xz, const void* conv_w, const void* conv_bias,
                    const void* x_proj, const void* dt_proj, const float* dt_bias, const float* a_log,
                    const float* skip, void* conv_state, float* ssm_state, const int32_t* in_slots,
                    const int32_t* out_slots, void* y, int64_t rows, int64_t n_slots, int64_t d_inner,
                    int64_t d_state, int64_t dt_rank, int64_t d_conv, ossm_stream_t stream_v) {
  clear_error();
  if (int rc = check_mixer("mixer_step", dtype, rows, rows, n_slots, d_inner, d_state, dt_rank, d_conv, ld_xz)) return rc;
  if (rows == 0 || d_inner == 0) return OSSM_OK;
  if (!xz || !conv_w || !x_proj || !dt_proj || !dt_bias || !a_log || !in_slots || !y ||
      (n_slots > 0 && (!ssm_state || (d_conv > 1 && !conv_state))))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, "mixer_step: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  StreamCall call(st);
  if (call.status()) return call.status();
  const auto run = [&](auto e) {
    return step(make<decltype(e)>(xz, ld_xz, conv_w, conv_bias, x_proj, dt_proj, dt_bias, a_log, skip, conv_state,
                                  ssm_state, in_slots, out_slots, nullptr, nullptr, y, rows, rows, n_slots, d_inner,
                                  d_state, dt_rank, d_conv), call, st);
  };
  return dtype == OSSM_BF16 ? run(bf16_t{}) : run(0.f);
}

int ossm_mixer_prompt(int dtype, const void* xz, int64_t ld_xz, const void* conv_w, const void* conv_bias,
                      const void* x_proj, const void* dt_proj, const float* dt_bias, const float* a_log,
                      const float* skip, void* conv_state, float* ssm_state, const int32_t* in_slots,
                      const int32_t* out_slots, const int32_t* offsets, const uint8_t* resume, void* y,
                      int64_t rows, int64_t n_seqs, int64_t n_slots, int64_t d_inner, int64_t d_state,
                      int64_t dt_rank, int64_t d_conv, ossm_stream_t stream_v) {
  clear_error();
  if (int rc = check_mixer("mixer_prompt", dtype, rows, n_seqs, n_slots, d_inner, d_state, dt_rank, d_conv, ld_xz)) return rc;
  if (d_inner == 0 || (rows == 0 && n_seqs == 0)) return OSSM_OK;
  if (n_seqs == 0) return set_error(OSSM_ERR_INVALID_ARGUMENT, "mixer_prompt: rows without a sequence");
  if ((rows > 0 && (!xz || !y)) || !conv_w || !x_proj || !dt_proj || !dt_bias || !a_log || !in_slots || !offsets ||
      (n_slots > 0 && (!ssm_state || (d_conv > 1 && !conv_state))))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, "mixer_prompt: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  StreamCall call(st);
  if (call.status()) return call.status();
  const auto run = [&](auto e) {
    return prompt(make<decltype(e)>(xz, ld_xz, conv_w, conv_bias, x_proj, dt_proj, dt_bias, a_log, skip, conv_state,
                                    ssm_state, in_slots, out_slots, offsets, resume, y, rows, n_seqs, n_slots, d_inner,
                                    d_state, dt_rank, d_conv), call, st);
  };
  return dtype == OSSM_BF16 ? run(bf16_t{}) : run(0.f);
}

}  // extern "C"
