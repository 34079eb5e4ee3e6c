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
// A token's launches: token_proj_kernel or token_tile_kernel (conv, its state's update,
// x_proj over a block of channels) and token_scan_kernel (the blocks' sums, dt, the state's update, the
// gate).  x_proj sums over all channels, so two launches is the least.
//
// A prompt batch is one row of packed tokens cut into chunks of equal length,
// whatever the prompts' lengths (the host never reads the offsets): a prompt's
// first token resets the recurrence, so a chunk may hold many prompts or a
// piece of one.  prompt_proj_kernel (conv and x_proj) and the first scan (dt_proj) put both
// projections on the matrix cores, u and p as three bf16 terms (split_mfma.hpp has
// the error).  mixer_scan_kernel<summary> finds what each chunk leaves to a zero
// carry and the sum of its dt (the decay over the chunk is exp(A sum dt)),
// the carry kernels fold the chunks in order, mixer_scan_kernel<output> walks the
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
#include "split_mfma.hpp"

namespace ossm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxConv = 8;
constexpr int kProjThreads = 256;
constexpr int kProjWaves = kProjThreads / kWave;
constexpr int kSub = 32;                       // channels of one wave's share of a token's x_proj
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
  float* part;   // [n_blocks][rows][Nc]: x_proj's sums over blocks (splits) of the channels
  float* u;      // tokens: [rows][Di]
  uint16_t* planes;  // prompts: [3][rows][Rp], the projections' part for dt
  float* bc;     // prompts: [rows][2][Npad], B and C, zero from N on
  float* dt;     // prompts: [rows][Di]
  float* local;  // prompts: [n_chunks][N][Di], a chunk's end from a zero carry
  float* carry;  // prompts: [n_chunks][N][Di], the state before a chunk
  float* sum_dt; // prompts: [n_chunks][Di], negative where a prompt starts in the chunk
  float* group_local;  // the same of groups of chunks: [n_groups][N][Di], [n_groups][Di]
  float* group_dt;
  float* init;   // prompts: [n_seqs][N][Di] copies of the resumed states, or null
  float* y_sum;  // prompts with N past a block of states: [rows][Di]
  long long ld;
  int rows, n_seqs, n_slots, Di, N, R, K, Nc, Npad, Rp, n_blocks, chunk, n_chunks, group, n_groups;
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

// Four consecutive elements.
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void load4(const bf16_t* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
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

// conv + SiLU of RB tokens over a block of channels, the conv's new state, and x_proj's
// partial sums over the block.  Each wave takes kSub of the channels and all Nc outputs, 64 at
// a time, one per lane; the waves' sums meet in LDS in a fixed order.  KT >= K taps.
template <class E, int RB, int KT>
__global__ __launch_bounds__(kProjThreads) void token_proj_kernel(Mixer<E> g, bool vec) {
  __shared__ float s_u[RB][kProjBlock];
  __shared__ float s_sum[kProjWaves][RB][kWave];
  const int blk = static_cast<int>(blockIdx.x % g.n_blocks);
  const int r0 = static_cast<int>(blockIdx.x / g.n_blocks) * RB;
  const int c0 = blk * kProjBlock;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = wave_id();
  const int skip_taps = KT - g.K;
  // every row's inputs are loaded before the first is used (a thread's rows are
  // kProjThreads / kProjBlock apart)
  constexpr int kRows = (RB * kProjBlock + kProjThreads - 1) / kProjThreads;
  const int c = tid % kProjBlock, d = min(c0 + c, g.Di - 1);
  float x[kRows][KT], wt[KT], v[kSub];
  const auto weights = [&](int j0) {
    const E* row = g.x_proj + static_cast<size_t>(min(j0 + lane, g.Nc - 1)) * g.Di;
#pragma unroll
    for (int q = 0; q < kSub; q += 8) {
      const int left = g.Di - (c0 + w * kSub + q);
      float e[8];
      load8(row + (left > 0 ? c0 + w * kSub + q : 0), left, vec, e);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[q + i] = e[i];
    }
  };
  weights(0);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = min(r0 + tid / kProjBlock + i * (kProjThreads / kProjBlock), g.rows - 1);
    const int slot = start_slot(g, r);
#pragma unroll
    for (int k = 0; k < KT - 1; ++k)
      x[i][k] = k >= skip_taps && slot >= 0
                    ? to_f(g.conv_state[(static_cast<size_t>(slot) * (g.K - 1) + k - skip_taps) * g.Di + d]) : 0.f;
    x[i][KT - 1] = to_f(g.xz[static_cast<size_t>(r) * g.ld + d]);
  }
#pragma unroll
  for (int k = 0; k < KT; ++k) wt[k] = k >= skip_taps ? to_f(g.conv_w[static_cast<size_t>(d) * g.K + k - skip_taps]) : 0.f;
  const float cb = g.conv_b != nullptr ? to_f(g.conv_b[d]) : 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int rr = tid / kProjBlock + i * (kProjThreads / kProjBlock), r = r0 + rr;
    if (rr >= RB) break;
    float u = 0.f;
    if (r < g.rows && c0 + c < g.Di) {
      float p = cb;
#pragma unroll
      for (int k = 0; k < KT; ++k)
        if (k >= skip_taps) p = fmaf(wt[k], x[i][k], p);
      u = silu_f(p);
      const int out = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[r];
      if (in_pool(g, out)) {
#pragma unroll
        for (int k = 1; k < KT; ++k)
          if (k > skip_taps)
            g.conv_state[(static_cast<size_t>(out) * (g.K - 1) + k - 1 - skip_taps) * g.Di + d] = from_f<E>(x[i][k]);
      }
      g.u[static_cast<size_t>(r) * g.Di + d] = u;
    }
    s_u[rr][c] = u;
  }
  __syncthreads();
  for (int j0 = 0; j0 < g.Nc; j0 += kWave) {
    float acc[RB], now[kSub];
#pragma unroll
    for (int i = 0; i < kSub; ++i) now[i] = v[i];
    if (j0 + kWave < g.Nc) weights(j0 + kWave);  // in flight under this step's sums
#pragma unroll
    for (int rr = 0; rr < RB; ++rr) {
      acc[rr] = 0.f;
#pragma unroll
      for (int i = 0; i < kSub; ++i) acc[rr] = fmaf(now[i], s_u[rr][w * kSub + i], acc[rr]);
    }
#pragma unroll
    for (int rr = 0; rr < RB; ++rr) s_sum[w][rr][lane] = acc[rr];
    __syncthreads();
    for (int i = tid; i < RB * kWave; i += kProjThreads) {
      const int rr = i / kWave, l = i % kWave;
      if (r0 + rr < g.rows && j0 + l < g.Nc) {
        float t = s_sum[0][rr][l];
#pragma unroll
        for (int q = 1; q < kProjWaves; ++q) t += s_sum[q][rr][l];
        g.part[(static_cast<size_t>(blk) * g.rows + r0 + rr) * g.Nc + j0 + l] = t;
      }
    }
    __syncthreads();
  }
}

// Column j of row r's projection, from the blocks' partial sums.
template <class E>
__device__ __forceinline__ float proj_of(const Mixer<E>& g, int r, int j) {
  const size_t step = static_cast<size_t>(g.rows) * g.Nc;
  const float* p = g.part + static_cast<size_t>(r) * g.Nc + j;
  float s = 0.f;
#pragma unroll 8
  for (int b = 0; b < g.n_blocks; ++b) s += p[b * step];
  return s;
}

// One token: a thread per channel, RB rows.  The first 16 states of all rows are asked
// for before the projections are summed: the states' traffic is what bounds a large
// batch, and this keeps 16 RB loads a thread in flight.  The rows' projections lie in LDS
// in three stretches padded with zeros, dt's to Rq, B's and C's to Nq (multiples of 16), so
// that four values come with a read.  VEC: A_log's and dt_proj's rows are whole 16-byte vectors.
template <class E, int RB, bool VEC>
__global__ __launch_bounds__(256) void token_scan_kernel(Mixer<E> g, int Rq, int Nq) {
  extern __shared__ __align__(16) float s_p[];  // [RB][Rq + 2 Nq]
  const int r0 = static_cast<int>(blockIdx.y) * RB;
  const int d_own = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x), d = min(d_own, g.Di - 1);
  constexpr int NB = 16;
  int in[RB], to[RB];
  float h[RB][NB], u[RB], z[RB], a2[NB];
#pragma unroll
  for (int rr = 0; rr < RB; ++rr) {
    const int r = min(r0 + rr, g.rows - 1);
    in[rr] = start_slot(g, r);
    to[rr] = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[r];
    const float* src = g.ssm + (static_cast<size_t>(max(in[rr], 0)) * g.N) * g.Di + d;
#pragma unroll
    for (int i = 0; i < NB; ++i) h[rr][i] = in[rr] >= 0 && i < g.N ? __builtin_nontemporal_load(src + static_cast<size_t>(i) * g.Di) : 0.f;
    u[rr] = g.u[static_cast<size_t>(r) * g.Di + d];
    z[rr] = to_f(g.xz[static_cast<size_t>(r) * g.ld + g.Di + d]);
  }
  const auto load_a = [&](int n0) {
    const float* p = g.a_log + static_cast<size_t>(d) * g.N + n0;
#pragma unroll
    for (int i = 0; i < NB; i += 4) {
      if (VEC && n0 + i + 4 <= g.N) {
        float q[4];
        load4(p + i, q);
#pragma unroll
        for (int k = 0; k < 4; ++k) a2[i + k] = q[k];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) a2[i + k] = n0 + i + k < g.N ? p[i + k] : 0.f;
      }
    }
  };
  load_a(0);
  // dt_proj's first 32 weights of the channel (zeros from R on)
  float wt[32];
  const auto load_w = [&](int q0) {
#pragma unroll
    for (int q = 0; q < 32; q += 8) {
      float e[8];
      load8(g.dt_proj + static_cast<size_t>(d) * g.R + (q0 + q < g.R ? q0 + q : 0), g.R - q0 - q, VEC, e);
#pragma unroll
      for (int i = 0; i < 8; ++i) wt[q + i] = e[i];
    }
  };
  load_w(0);
  const int width = Rq + 2 * Nq;
  for (int i = threadIdx.x; i < RB * width; i += blockDim.x) {
    const int rr = i / width, k = i % width, c = k - Rq, second = c >= Nq ? 1 : 0, n = c - second * Nq;
    const int j = k < Rq ? (k < g.R ? k : -1) : (n < g.N ? g.R + second * g.N + n : -1);
    s_p[i] = j >= 0 && r0 + rr < g.rows ? proj_of(g, r0 + rr, j) : 0.f;
  }
  __syncthreads();
  float dt[RB];
  const float bias = g.dt_bias[d];
#pragma unroll
  for (int rr = 0; rr < RB; ++rr) dt[rr] = bias;
  for (int q0 = 0; q0 < g.R; q0 += 32) {
    if (q0 > 0) load_w(q0);
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      if (q0 + i < g.R) {  // (what a zero weight meets is a zero)
#pragma unroll
        for (int rr = 0; rr < RB; ++rr) {
          const float4 p = *reinterpret_cast<const float4*>(s_p + rr * width + q0 + i);
          dt[rr] = fmaf(wt[i + 3], p.w, fmaf(wt[i + 2], p.z, fmaf(wt[i + 1], p.y, fmaf(wt[i], p.x, dt[rr]))));
        }
      }
    }
  }
  if (d_own >= g.Di) return;
  const float skip = g.skip != nullptr ? g.skip[d] : 0.f;
  float y[RB], du[RB];
#pragma unroll
  for (int rr = 0; rr < RB; ++rr) {
    dt[rr] = softplus_f(dt[rr]);
    du[rr] = dt[rr] * u[rr];
    y[rr] = skip * u[rr];
  }
  for (int n0 = 0; n0 < g.N; n0 += NB) {
    if (n0 > 0) load_a(n0);
#pragma unroll
    for (int i = 0; i < NB; ++i) a2[i] = -expf(a2[i]) * kLog2e;
#pragma unroll
    for (int rr = 0; rr < RB; ++rr) {
      if (n0 > 0) {
        const float* src = g.ssm + (static_cast<size_t>(max(in[rr], 0)) * g.N + n0) * g.Di + d;
#pragma unroll
        for (int i = 0; i < NB; ++i) h[rr][i] = in[rr] >= 0 && n0 + i < g.N ? src[static_cast<size_t>(i) * g.Di] : 0.f;
      }
      const float* B = s_p + rr * width + Rq + n0;
      const bool keep = r0 + rr < g.rows && in_pool(g, to[rr]);
      float* dst = g.ssm + (static_cast<size_t>(keep ? to[rr] : 0) * g.N + n0) * g.Di + d;
#pragma unroll
      for (int i = 0; i < NB; i += 4) {
        float b[4], c[4];
        load4(B + i, b);
        load4(B + Nq + i, c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float v = fmaf(__builtin_amdgcn_exp2f(a2[i + k] * dt[rr]), h[rr][i + k], du[rr] * b[k]);
          if (n0 + i + k < g.N) {
            y[rr] = fmaf(c[k], v, y[rr]);
            if (keep) __builtin_nontemporal_store(v, dst + static_cast<size_t>(i + k) * g.Di);
          }
        }
      }
    }
  }
#pragma unroll
  for (int rr = 0; rr < RB; ++rr)
    if (r0 + rr < g.rows) {
      const bool padding = in[rr] < 0 && !in_pool(g, to[rr]);
      g.y[static_cast<size_t>(r0 + rr) * g.Di + d] = from_f<E>(padding ? 0.f : y[rr] * silu_f(z[rr]));
    }
}

// ---- prompts: the projections on the matrix cores -----------------------------------

// x as the three bf16 terms of split_mfma.hpp, two values to a word; one that is not
// finite as (x, 0, 0), one that would round past the largest bf16 as that and the rest.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&t)[3]) {
  constexpr float kTop = 3.3895313892515355e38f;  // the largest bf16
  const bool fa = fabsf(a) <= 3.4028234663852886e38f, fb = fabsf(b) <= 3.4028234663852886e38f;
  t[0] = pack_bf16(fa ? fminf(fmaxf(a, -kTop), kTop) : a, fb ? fminf(fmaxf(b, -kTop), kTop) : b);
  const float ra = fa ? a - bf16_lo(t[0]) : 0.f, rb = fb ? b - bf16_hi(t[0]) : 0.f;
  t[1] = pack_bf16(ra, rb);
  t[2] = pack_bf16(ra - bf16_lo(t[1]), rb - bf16_hi(t[1]));
}

// Rows of `width` (a multiple of 64) bf16 in LDS, in 16-byte chunks: chunk c of row r
// sits at c ^ (r % 8), which spreads a fragment's rows over the banks.
__device__ __forceinline__ int plane_at(int r, int k, int width) { return r * width + (((k >> 3) ^ (r & 7)) << 3) + (k & 7); }

// A weight's fragment: eight values from k of row j, as its terms (zeros past the row).
template <class E>
struct Weight8;
template <>
struct Weight8<bf16_t> {
  bf16x8 t[1];
  __device__ __forceinline__ void load(const bf16_t* row, int k, int n, bool vec) {
    if (vec && k + 8 <= n) {
      t[0] = *reinterpret_cast<const bf16x8*>(row + k);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[0][i] = __builtin_bit_cast(__bf16, k + i < n ? row[k + i].bits : static_cast<uint16_t>(0));
    }
  }
  __device__ __forceinline__ void split() {}
};
template <>
struct Weight8<float> {
  float x[8];
  bf16x8 t[3];
  __device__ __forceinline__ void load(const float* row, int k, int n, bool vec) { load8(row + (k < n ? k : 0), n - k, vec, x); }
  __device__ __forceinline__ void split() {
    const SplitFrag f = split8(x);
    t[0] = f.t0;
    t[1] = f.t1;
    t[2] = f.t2;
  }
};

// c += a b over 16 k, the terms of order up to two, smallest first (a bf16 weight is one term)
__device__ __forceinline__ floatx16 mfma_terms(const bf16x8 (&a)[3], const Weight8<bf16_t>& b, floatx16 c) {
  c = mfma_bf16(a[2], b.t[0], c);
  c = mfma_bf16(a[1], b.t[0], c);
  return mfma_bf16(a[0], b.t[0], c);
}
__device__ __forceinline__ floatx16 mfma_terms(const bf16x8 (&a)[3], const Weight8<float>& b, floatx16 c) {
  return mfma_split(SplitFrag{a[0], a[1], a[2]}, SplitFrag{b.t[0], b.t[1], b.t[2]}, c);
}

// The sums of the second way wherever the first's are not finite.
__device__ __forceinline__ void keep_finite(floatx16 (&acc)[2], const floatx16 (&first)[2]) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[j][r] = fabsf(first[j][r]) <= 3.4028234663852886e38f ? first[j][r] : acc[j][r];
}

// The three terms of an LDS plane set at (r, k), added up again.
__device__ __forceinline__ float planes_sum(const uint16_t* s, int plane, int at) {
  return (to_f(bf16_t{s[2 * plane + at]}) + to_f(bf16_t{s[plane + at]})) + to_f(bf16_t{s[at]});
}

// Eight consecutive elements, on a 16-byte boundary.
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

constexpr int kTileRows = 32, kTileK = 128;  // token_tile_kernel's
constexpr int kTileThreads = kTileRows * kTileK / 8;

// token_proj_kernel for many rows of whole vectors: a tile of 32 sequences and 128 channels, a
// thread 8 channels of a sequence, x_proj on the matrix cores, a wave 32 of its outputs at a
// time over half of the channels.  All of it is asked for before the first barrier; latency
// bounds it (8 us of a step of 256 sequences, 17 by token_proj_kernel).
template <class E, int KT>
__global__ __launch_bounds__(kTileThreads, 2) void token_tile_kernel(Mixer<E> g) {
  __shared__ __align__(16) uint16_t s_u[3 * kTileRows * kTileK];
  __shared__ float s_half[4][16][kWave];
  constexpr int kSteps = kTileK / 32;  // a wave's k steps
  constexpr int kPlane = kTileRows * kTileK;
  const int blk = static_cast<int>(blockIdx.x % g.n_blocks), c0 = blk * kTileK;
  const int r0 = static_cast<int>(blockIdx.x / g.n_blocks) * kTileRows;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), l32 = lane & 31, half = lane >> 5;
  const int w = wave_id() & 3, kh = wave_id() >> 2, kb = kh * (kTileK / 2);  // the wave's outputs, its half of the channels
  constexpr int kChunks = kTileK / 8;
  const int row = tid / kChunks, r = min(r0 + row, g.rows - 1), ch = c0 + tid % kChunks * 8, d = min(ch, g.Di - 8);
  const bool live = r0 + row < g.rows && ch < g.Di;
  const int skip_taps = KT - g.K;
  Weight8<E> wt[kSteps];
  const auto weights = [&](int j0) {
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk)
      wt[kk].load(g.x_proj + static_cast<size_t>(min(j0 + l32, g.Nc - 1)) * g.Di, c0 + kb + kk * 16 + half * 8, g.Di, true);
  };
  weights(w * 32);
  const int slot = start_slot(g, r), to = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[r];
  float x[KT][8], cw[KT][8], u[8];
#pragma unroll
  for (int k = 0; k < KT - 1; ++k) {
    if (k >= skip_taps && slot >= 0) {
      load8(g.conv_state + (static_cast<size_t>(slot) * (g.K - 1) + k - skip_taps) * g.Di + d, 8, true, x[k]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
    }
  }
  load8(g.xz + static_cast<size_t>(r) * g.ld + d, 8, true, x[KT - 1]);
  if (KT == 4 && g.K == 4) {  // a channel's taps side by side: two channels to eight
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float q[8];
      load8(g.conv_w + static_cast<size_t>(d + e) * 4, 8, true, q);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        cw[k % KT][e] = q[k];
        cw[k % KT][e + 1] = q[4 + k];
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) cw[k][e] = k >= skip_taps ? to_f(g.conv_w[static_cast<size_t>(d + e) * g.K + k - skip_taps]) : 0.f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = 0.f;
  if (g.conv_b != nullptr) load8(g.conv_b + d, 8, true, u);
#pragma unroll
  for (int k = 0; k < KT; ++k)
    if (k >= skip_taps)
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = fmaf(cw[k][e], x[k][e], u[e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = live ? silu_f(u[e]) : 0.f;
  uint32_t t[4][3];
#pragma unroll
  for (int e = 0; e < 4; ++e) split_pair(u[2 * e], u[2 * e + 1], t[e]);
#pragma unroll
  for (int q = 0; q < 3; ++q)
    *reinterpret_cast<uint4*>(&s_u[q * kPlane + plane_at(row, tid % kChunks * 8, kTileK)]) = make_uint4(t[0][q], t[1][q], t[2][q], t[3][q]);
  if (live) {
    store8(g.u + static_cast<size_t>(r) * g.Di + d, u);
    if (in_pool(g, to)) {
#pragma unroll
      for (int k = 1; k < KT; ++k)
        if (k > skip_taps) store8(g.conv_state + (static_cast<size_t>(to) * (g.K - 1) + k - 1 - skip_taps) * g.Di + d, x[k]);
    }
  }
  __syncthreads();
  for (int base = 0; base < g.Nc; base += 128) {
    const int j0 = base + w * 32;
    if (base > 0) weights(j0);
    floatx16 acc[2] = {};  // (the second stays zero)
    if (j0 < g.Nc) {
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk) {
        bf16x8 a[3];
#pragma unroll
        for (int q = 0; q < 3; ++q)
          a[q] = *reinterpret_cast<const bf16x8*>(&s_u[q * kPlane + plane_at(l32, kb + kk * 16 + half * 8, kTileK)]);
        wt[kk].split();
        acc[0] = mfma_terms(a, wt[kk], acc[0]);
      }
      if (any_nonfinite(acc)) {
        floatx16 again[2] = {};
        const E* row_w = g.x_proj + static_cast<size_t>(min(j0 + l32, g.Nc - 1)) * g.Di;
#pragma unroll 1
        for (int q = 0; q < kTileK / 2; q += 2) {
          const int k = kb + q + half;
          again[0] = mfma32(planes_sum(s_u, kPlane, plane_at(l32, k, kTileK)), c0 + k < g.Di ? to_f(row_w[c0 + k]) : 0.f, again[0]);
        }
        keep_finite(again, acc);
        acc[0] = again[0];
      }
    }
    if (base > 0) __syncthreads();
    if (kh == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s_half[w][i][lane] = acc[0][i];
    }
    __syncthreads();
    if (kh == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = r0 + 8 * (i >> 2) + 4 * half + (i & 3), col = j0 + l32;
        if (at < g.rows && col < g.Nc)
          g.part[(static_cast<size_t>(blk) * g.rows + at) * g.Nc + col] = acc[0][i] + s_half[w][i][lane];
      }
    }
  }
}

constexpr int kPtRows = 64, kPtK = 64, kPtCols = 128;  // prompt_proj_kernel's tile and k step

// A thread's share of a tile's conv: 4 channels of 4 rows, and the rows before them.
// VEC: whole quads of channels, on 4-element boundaries.
template <class E, int KT, bool VEC>
struct ConvShare {
  float x[4 + KT - 1][4], w[4][KT], b[4];

  __device__ __forceinline__ void load(const Mixer<E>& g, int r_first, int d0) {
    const int skip_taps = KT - g.K;
    const int dv = VEC ? min(d0, g.Di - 4) : d0;
#pragma unroll
    for (int i = 0; i < 4 + KT - 1; ++i) {
      const E* row = g.xz + static_cast<size_t>(min(max(r_first - (KT - 1) + i, 0), g.rows - 1)) * g.ld;
      if constexpr (VEC) {
        load4(row + dv, x[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = to_f(row[min(d0 + e, g.Di - 1)]);
      }
    }
    if (VEC && KT == 4 && g.K == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float q[4];
        load4(g.conv_w + static_cast<size_t>(dv + e) * 4, q);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[e][k] = q[k];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int k = 0; k < KT; ++k)
          w[e][k] = k >= skip_taps ? to_f(g.conv_w[static_cast<size_t>(min(d0 + e, g.Di - 1)) * g.K + k - skip_taps]) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = g.conv_b != nullptr ? to_f(g.conv_b[min(d0 + e, g.Di - 1)]) : 0.f;
  }

  // u of the rows in `inside` (bit r: row r of the tile and the K - 1 before it are one
  // prompt's), zeros for the rows in `padding`, as three planes in LDS
  __device__ __forceinline__ void store(const Mixer<E>& g, int rr0, int quad, int d0, uint64_t inside, uint64_t padding,
                                        uint16_t* s_u) const {
    const int skip_taps = KT - g.K;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = rr0 + i;
      float u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = b[e];
#pragma unroll
      for (int k = 0; k < KT; ++k)
        if (k >= skip_taps)
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = fmaf(w[e][k], x[i + k][e], u[e]);
      const bool zero = (padding >> rr) & 1;
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = d0 + e < g.Di && !zero ? silu_f(u[e]) : 0.f;
      uint32_t t0[3], t1[3];
      split_pair(u[0], u[1], t0);
      split_pair(u[2], u[3], t1);
      const int at = plane_at(rr, 4 * quad, kPtK);
      if (((inside | padding) >> rr) & 1) {
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<uint2*>(&s_u[q * (kPtRows * kPtK) + at]) = make_uint2(t0[q], t1[q]);
      }
    }
  }
};

// The other rows of the tile, a prompt's first K - 1: a wave a row, a lane a channel.
template <class E>
__device__ __forceinline__ void store_first_rows(const Mixer<E>& g, int r0, int k0, uint64_t others, const int* s_start,
                                                 const int* s_slot, uint16_t* s_u) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), d = min(k0 + lane, g.Di - 1);
  int turn = 0;
#pragma unroll 1
  for (; others != 0; others &= others - 1, ++turn) {
    if ((turn & 3) != wave_id()) continue;
    const int rr = __builtin_ctzll(others), start = s_start[rr], slot = s_slot[rr];
    float p = g.conv_b != nullptr ? to_f(g.conv_b[d]) : 0.f;
#pragma unroll 1
    for (int k = 0; k < g.K; ++k)
      p = fmaf(to_f(g.conv_w[static_cast<size_t>(d) * g.K + k]), conv_input(g, r0 + rr - (g.K - 1) + k, start, slot, d), p);
    uint32_t t[3];
    split_pair(k0 + lane < g.Di ? silu_f(p) : 0.f, 0.f, t);
    const int at = plane_at(rr, lane, kPtK);
#pragma unroll
    for (int q = 0; q < 3; ++q) s_u[q * (kPtRows * kPtK) + at] = static_cast<uint16_t>(t[q]);
  }
}

// Conv + SiLU of a tile of kPtRows tokens, kPtK channels at a time, and x_proj's sums over
// this split's channels for kPtCols of the Nc outputs.  u goes from registers into LDS as
// three bf16 planes; a wave takes 32 rows and 64 outputs, the weights' fragments straight
// from memory (all workgroups read the same few hundred kB).  Sums that are not
// finite (a term of an infinite weight against a zero one) are formed again on the
// fp32 instruction; finite ones stay as they are, whatever their neighbours.
template <class E, int KT, bool VEC>
__global__ __launch_bounds__(256, 2) void prompt_proj_kernel(Mixer<E> g, int per_split, bool vec) {
  __shared__ __align__(16) uint16_t s_u[3 * kPtRows * kPtK];
  __shared__ int s_start[kPtRows], s_slot[kPtRows];
  __shared__ uint64_t s_rows[2];  // rows inside a prompt, rows of padding
  const int groups = (g.Nc + kPtCols - 1) / kPtCols;
  int id = static_cast<int>(blockIdx.x);
  const int col0 = id % groups * kPtCols;
  id /= groups;
  const int split = id % g.n_blocks, r0 = id / g.n_blocks * kPtRows;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = wave_id();
  const int quad = tid & 15, rr0 = (tid >> 4) * 4;  // the conv's share: 4 channels of 4 rows
  const int rf = (w & 1) * 32, cf = col0 + (w >> 1) * 64;  // the product's: 32 rows, 64 outputs
  const int l32 = lane & 31, half = lane >> 5;
  const int k_first = split * per_split, k_end = min(g.Di, k_first + per_split);
  ConvShare<E, KT, VEC> conv;
  conv.load(g, r0 + rr0, k_first + 4 * quad);
  if (tid < kPtRows) {
    const int r = r0 + tid;
    int start = INT_MAX, slot = -1;  // INT_MAX: padding
    if (r < g.rows) {
      const int s = seq_of(g, r);
      if (s >= 0 && r < offset_of(g, s + 1)) { start = offset_of(g, s); slot = start_slot(g, s); }
    }
    s_start[tid] = start;
    s_slot[tid] = slot;
    const uint64_t inside = __ballot(start != INT_MAX && r - (g.K - 1) >= start), padding = __ballot(start == INT_MAX);
    if (tid == 0) { s_rows[0] = inside; s_rows[1] = padding; }
  }
  __syncthreads();
  const uint64_t inside = s_rows[0], padding = s_rows[1];
  const E* rows_w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) rows_w[j] = g.x_proj + static_cast<size_t>(min(cf + j * 32 + l32, g.Nc - 1)) * g.Di;
  const bool idle = cf >= g.Nc;  // a wave without outputs
  floatx16 acc[2] = {};
  for (int k0 = k_first; k0 < k_end; k0 += kPtK) {
    __syncthreads();  // the last step's products have read s_u
    Weight8<E> wt[kPtK / 16][2];
    if (!idle) {
#pragma unroll
      for (int kk = 0; kk < kPtK / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 2; ++j) wt[kk][j].load(rows_w[j], k0 + kk * 16 + half * 8, g.Di, vec);
    }
    conv.store(g, rr0, quad, k0 + 4 * quad, inside, padding, s_u);
    store_first_rows(g, r0, k0, ~(inside | padding), s_start, s_slot, s_u);
    if (k0 + kPtK < k_end) conv.load(g, r0 + rr0, k0 + kPtK + 4 * quad);  // in flight under the products
    __syncthreads();
    if (!idle) {
#pragma unroll
      for (int kk = 0; kk < kPtK / 16; ++kk) {
        bf16x8 a[3];
#pragma unroll
        for (int q = 0; q < 3; ++q)
          a[q] = *reinterpret_cast<const bf16x8*>(&s_u[q * (kPtRows * kPtK) + plane_at(rf + l32, kk * 16 + half * 8, kPtK)]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          wt[kk][j].split();
          acc[j] = mfma_terms(a, wt[kk][j], acc[j]);
        }
      }
    }
  }
  if (__syncthreads_or(any_nonfinite(acc))) {
    floatx16 again[2] = {};
#pragma unroll 1
    for (int k0 = k_first; k0 < k_end; k0 += kPtK) {
      conv.load(g, r0 + rr0, k0 + 4 * quad);
      __syncthreads();
      conv.store(g, rr0, quad, k0 + 4 * quad, inside, padding, s_u);
      store_first_rows(g, r0, k0, ~(inside | padding), s_start, s_slot, s_u);
      __syncthreads();
#pragma unroll 1
      for (int q = 0; q < kPtK; q += 2) {
        const int k = q + half;
        const float a = planes_sum(s_u, kPtRows * kPtK, plane_at(rf + l32, k, kPtK));
#pragma unroll
        for (int j = 0; j < 2; ++j) again[j] = mfma32(a, k0 + k < g.Di ? to_f(rows_w[j][k0 + k]) : 0.f, again[j]);
      }
    }
    keep_finite(again, acc);
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[j] = again[j];
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = r0 + rf + 8 * (r >> 2) + 4 * half + (r & 3), col = cf + j * 32 + l32;
      if (row < g.rows && col < g.Nc) g.part[(static_cast<size_t>(split) * g.rows + row) * g.Nc + col] = acc[j][r];
    }
}

// Prompt s's last K - 1 inputs, and its state where it is empty.
template <class E>
__device__ __forceinline__ void finish(const Mixer<E>& g, int d, int s) {
  if (d >= g.Di) return;
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
  if (start == end && to != slot) {
    const float* src = g.ssm + (static_cast<size_t>(max(slot, 0)) * g.N) * g.Di + d;
    float* dst = g.ssm + (static_cast<size_t>(to) * g.N) * g.Di + d;
    for (int n0 = 0; n0 < g.N; n0 += 16) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = slot >= 0 ? src[static_cast<size_t>(min(n0 + i, g.N - 1)) * g.Di] : 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (n0 + i < g.N) dst[static_cast<size_t>(n0 + i) * g.Di] = v[i];
    }
  }
}

template <class E>
__global__ __launch_bounds__(256) void mixer_finish_kernel(Mixer<E> g) {
  finish(g, static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x), static_cast<int>(blockIdx.y));
}

// x_proj's sums over its splits: B and C in float32, the part for dt as three bf16 planes
// [3][rows][Rp] (zeros from R on).  Workgroups from `sums` on finish the prompts, where
// nothing is resumed: no later kernel then reads what they write.
template <class E>
__global__ __launch_bounds__(256) void prompt_sum_kernel(Mixer<E> g, unsigned sums) {
  if (blockIdx.x >= sums) {
    const int blocks = (g.Di + 255) / 256, id = static_cast<int>(blockIdx.x - sums);
    finish(g, id % blocks * 256 + static_cast<int>(threadIdx.x), id / blocks);
    return;
  }
  const int cols = g.Rp + 2 * g.Npad;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<long long>(g.rows) * cols) return;
  const int r = static_cast<int>(i / cols), k = static_cast<int>(i % cols);
  const size_t plane = static_cast<size_t>(g.rows) * g.Rp;
  if (k < g.Rp) {
    uint32_t t[3];
    split_pair(k < g.R ? proj_of(g, r, k) : 0.f, 0.f, t);
#pragma unroll
    for (int q = 0; q < 3; ++q) g.planes[q * plane + static_cast<size_t>(r) * g.Rp + k] = static_cast<uint16_t>(t[q]);
  } else {
    const int c = k - g.Rp, second = c >= g.Npad ? 1 : 0, n = c - second * g.Npad;
    g.bc[static_cast<size_t>(r) * 2 * g.Npad + c] = n < g.N ? proj_of(g, r, g.R + second * g.N + n) : 0.f;
  }
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
constexpr int kGroup = 4;   // tokens whose inputs are loaded together
constexpr int kStage = 32;  // tokens whose B and C are in LDS

// dt_proj's sums of 32 tokens (from r0) and the wave's 64 channels (from cw), both operands'
// fragments straight from memory: the planes and the weights are read from the caches by
// every tile.  Register r of lane l: token 8 (r / 4) + 4 (l / 32) + r % 4, channel l % 32
// of each half.
template <class E>
__device__ __forceinline__ void dt_sums(const Mixer<E>& g, int r0, int cw, bool vec, floatx16 (&acc)[2]) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), l32 = lane & 31, half = lane >> 5;
  const size_t plane = static_cast<size_t>(g.rows) * g.Rp;
  const uint16_t* row = g.planes + static_cast<size_t>(min(r0 + l32, g.rows - 1)) * g.Rp;
  const E* rows_w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    rows_w[j] = g.dt_proj + static_cast<size_t>(min(cw + j * 32 + l32, g.Di - 1)) * g.R;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[j][r] = 0.f;
  }
  constexpr int kAhead = 2;  // k steps whose fragments are asked for together
#pragma unroll 1
  for (int k0 = 0; k0 < g.Rp; k0 += 16 * kAhead) {
    bf16x8 a[kAhead][3];
    Weight8<E> wt[kAhead][2];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int k = min(k0 + q * 16, g.Rp - 16) + half * 8;
#pragma unroll
      for (int t = 0; t < 3; ++t) a[q][t] = *reinterpret_cast<const bf16x8*>(row + t * plane + k);
#pragma unroll
      for (int j = 0; j < 2; ++j) wt[q][j].load(rows_w[j], k, g.R, vec);
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (k0 + q * 16 < g.Rp) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          wt[q][j].split();
          acc[j] = mfma_terms(a[q], wt[q][j], acc[j]);
        }
      }
  }
  if (any_nonfinite(acc)) {
    floatx16 again[2] = {};
#pragma unroll 1
    for (int k0 = 0; k0 < g.Rp; k0 += 2) {
      const int k = k0 + half;
      const float a = (to_f(bf16_t{row[2 * plane + k]}) + to_f(bf16_t{row[plane + k]})) + to_f(bf16_t{row[k]});
#pragma unroll
      for (int j = 0; j < 2; ++j) again[j] = mfma32(a, k < g.R ? to_f(rows_w[j][k]) : 0.f, again[j]);
    }
    keep_finite(again, acc);
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[j] = again[j];
  }
}

constexpr int kDtRows = 32, kDtCols = 256;  // prompt_dt_kernel's tile, a wave 32 x 64 of it

// dt of a batch large enough to fill the card without the scans' help.  Many small waves:
// weights kept in registers over several tiles cost the occupancy that hides the loads
// (75 us against 68 at [16384, 2048], whose write alone takes 27).
template <class E>
__global__ __launch_bounds__(256, 4) void prompt_dt_kernel(Mixer<E> g, bool vec) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), l32 = lane & 31, half = lane >> 5;
  const int r0 = static_cast<int>(blockIdx.x) * kDtRows;
  const int cw = static_cast<int>(blockIdx.y) * kDtCols + wave_id() * 64;
  if (cw >= g.Di) return;  // no barriers below
  float bias[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) bias[j] = g.dt_bias[min(cw + j * 32 + l32, g.Di - 1)];
  floatx16 acc[2];
  dt_sums(g, r0, cw, vec, acc);
  const bool whole = r0 + kDtRows <= g.rows;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int d = cw + j * 32 + l32;
    if (d >= g.Di) continue;
    float* out = g.dt + static_cast<size_t>(r0) * g.Di + d;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int at = 8 * (r >> 2) + 4 * half + (r & 3);
      const float v = softplus_f(acc[j][r] + bias[j]);
      if (whole || r0 + at < g.rows) out[static_cast<size_t>(at) * g.Di] = v;
    }
  }
}

// One thread per channel walks a chunk, NB states (from n_base) in registers and KT conv
// taps (those before the last K are skipped).  OUT: from the chunk's carry, writing y and
// the states of the prompts that end here; else from the last prompt start in the chunk
// (or a zero carry), leaving the chunk's end and its sum of dt.
//
// Bound by the VALU: a token and channel take about 40 instructions, a state 5, one of
// them an exponential of four issue slots.  B and C, the same for all channels, come from
// LDS by broadcast reads, a stage of tokens at a time: as scalar loads they were
// waited for token by token, 0.8 us each where few waves run.
//
// DT: this pass forms dt of its stages on the matrix cores (the first of the passes, where
// the chunks leave the card half empty) and, where another follows, leaves it in memory.
template <class E, int NB, int KT, bool OUT, bool DT>
__global__ __launch_bounds__(kScanThreads, NB <= 16 ? (DT ? 3 : 4) : 2) void mixer_scan_kernel(Mixer<E> g, int n_base, bool vec) {
  __shared__ __align__(16) float s_bc[kStage][2 * NB];
  __shared__ float s_dt[DT ? kStage : 1][DT ? kScanThreads : 1];
  const int d_own = static_cast<int>(blockIdx.x) * kScanThreads + static_cast<int>(threadIdx.x);
  const bool live = d_own < g.Di;
  const int d = min(d_own, g.Di - 1);
  const int c = static_cast<int>(blockIdx.y);
  const int t0 = c * g.chunk, t1 = min(t0 + g.chunk, g.rows);
  const bool last_block = n_base + NB >= g.N;
  float a2[NB], h[NB], cw[KT], win[KT];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    a2[i] = n_base + i < g.N ? -expf(g.a_log[static_cast<size_t>(d) * g.N + n_base + i]) * kLog2e : 0.f;
    h[i] = 0.f;
  }
  const int skip_taps = KT - g.K;
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    cw[k] = k >= skip_taps ? to_f(g.conv_w[static_cast<size_t>(d) * g.K + k - skip_taps]) : 0.f;
    win[k] = 0.f;
  }
  const float cb = g.conv_b != nullptr ? to_f(g.conv_b[d]) : 0.f;
  const float skip = g.skip != nullptr ? g.skip[d] : 0.f;

  int s = seq_of(g, OUT ? t0 : t1 - 1);
  int t = t0;
  float dt_sum = 0.f;
  if constexpr (!OUT) {
    // (none: padding only, and the next chunk starts a prompt)
    const int start = s >= 0 ? offset_of(g, s) : t1;
    if (start >= t0) { t = start; dt_sum = -1.f; }
    if (c + 1 == g.n_chunks) t = t1;  // nothing follows: it needs no summary
  }
  bool begun = false;  // h and the window are sequence s's at t
#pragma unroll 1
  for (int b0 = t0; b0 < t1; b0 += kStage) {
    const int b1 = min(b0 + kStage, t1);
    if (!DT && t >= b1) continue;  // (the same for the whole workgroup)
    __syncthreads();
    if constexpr (DT) {
      const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), l32 = lane & 31, half = lane >> 5, w = wave_id();
      const int cw = static_cast<int>(blockIdx.x) * kScanThreads + w * kWave;
      floatx16 acc[2];
      dt_sums(g, b0, cw, vec, acc);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int ch = cw + j * 32 + l32;
        const float bias = g.dt_bias[min(ch, g.Di - 1)];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = 8 * (r >> 2) + 4 * half + (r & 3);
          const float v = softplus_f(acc[j][r] + bias);
          s_dt[row][w * kWave + j * 32 + l32] = v;
          if (g.dt != nullptr && ch < g.Di && b0 + row < b1) g.dt[static_cast<size_t>(b0 + row) * g.Di + ch] = v;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kStage * 2 * NB / 4 / kScanThreads + 1; ++q) {
      const int i = (q * kScanThreads + static_cast<int>(threadIdx.x)) * 4;
      const int row = i / (2 * NB), k = i % (2 * NB);
      if (row < kStage && b0 + row < t1) {
        const float* src = g.bc + static_cast<size_t>(b0 + row) * 2 * g.Npad + n_base + (k < NB ? k : g.Npad + k - NB);
        *reinterpret_cast<float4*>(&s_bc[row][k]) = *reinterpret_cast<const float4*>(src);
      }
    }
    __syncthreads();
    while (t < b1) {
      // the segment [t, e) of sequence s in this stage
      if (s < 0 || t >= offset_of(g, s + 1)) {  // padding
        const int e = s + 1 < g.n_seqs ? min(b1, max(offset_of(g, s + 1), t + 1)) : b1;
        if constexpr (OUT)
          if (last_block && live)
            for (int i = t; i < e; ++i) g.y[static_cast<size_t>(i) * g.Di + d] = from_f<E>(0.f);
        t = e;
      } else {
        const int start = offset_of(g, s), end = offset_of(g, s + 1), e = min(b1, end);
        if (!begun) {
          begun = true;
          const int slot = start_slot(g, s);
          const bool first = t == start, carried = OUT && !first && t == t0 && c > 0;
          const float* src = first ? (g.init != nullptr ? g.init + (static_cast<size_t>(s) * g.N) * g.Di
                                                        : g.ssm + (static_cast<size_t>(max(slot, 0)) * g.N) * g.Di)
                                   : g.carry + (static_cast<size_t>(c) * g.N) * g.Di;
          const bool any = first ? slot >= 0 : carried;
#pragma unroll
          for (int i = 0; i < NB; ++i)
            h[i] = any && n_base + i < g.N ? src[static_cast<size_t>(n_base + i) * g.Di + d] : 0.f;
#pragma unroll
          for (int k = 0; k < KT - 1; ++k)
            win[k] = k >= skip_taps ? conv_input(g, t - (KT - 1) + k, start, slot, d) : 0.f;
        }
#pragma unroll 1
        for (; t < e; t += kGroup) {
          float x[kGroup], z[kGroup], dt[kGroup], ys[kGroup];
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            const size_t r = static_cast<size_t>(min(t + i, e - 1));
            x[i] = to_f(g.xz[r * g.ld + d]);
            dt[i] = DT ? s_dt[min(t + i, e - 1) - b0][threadIdx.x] : g.dt[r * g.Di + d];
            if constexpr (OUT) {
              z[i] = to_f(g.xz[r * g.ld + g.Di + d]);
              ys[i] = n_base > 0 ? g.y_sum[r * g.Di + d] : 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            if (t + i >= e) break;
            __builtin_amdgcn_sched_barrier(0);  // a token's B and C are read with it, not the group's at once
            const float* B = s_bc[t + i - b0];
            float p = cb;
#pragma unroll
            for (int k = 0; k < KT - 1; ++k)
              if (k >= skip_taps) p = fmaf(cw[k], win[k], p);
            p = fmaf(cw[KT - 1], x[i], p);
#pragma unroll
            for (int k = 0; k + 1 < KT - 1; ++k) win[k] = win[k + 1];
            win[KT - 2] = x[i];
            const float u = silu_f(p);
            const float du = dt[i] * u;
            float y = OUT && n_base == 0 ? skip * u : ys[i];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const float decay = __builtin_amdgcn_exp2f(a2[n] * dt[i]);
              h[n] = fmaf(decay, h[n], du * B[n]);
              if constexpr (OUT) y = fmaf(B[NB + n], h[n], y);
            }
            if constexpr (OUT) {
              const size_t at = static_cast<size_t>(t + i) * g.Di + d;
              if (live) {
                if (last_block) g.y[at] = from_f<E>(y * silu_f(z[i]));
                else g.y_sum[at] = y;
              }
            } else if (dt_sum >= 0.f) {
              dt_sum += dt[i];
            }
          }
        }
        t = e;
        if (e == end) {
          begun = false;
          if constexpr (OUT) {
            const int to = (g.out_slots != nullptr ? g.out_slots : g.in_slots)[s];
            if (in_pool(g, to) && live) {
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
  }
  if constexpr (!OUT) {
    if (!live) return;
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (n_base + i < g.N) g.local[(static_cast<size_t>(c) * g.N + n_base + i) * g.Di + d] = h[i];
    if (n_base == 0) g.sum_dt[static_cast<size_t>(c) * g.Di + d] = dt_sum;
  }
}

constexpr int kCarryAhead = 16;  // chunks whose summaries are loaded together

// h after a chunk that ends at `local` from zero, its sum of dt `sum`: the transition
// exp(A sum) in two halves, since it may underflow where its product with the state does
// not (1e33 under e^-96), and each at least the smallest normal number, since an infinite
// state stays infinite under every decay (what that adds to a finite one is below 2^-124).
__device__ __forceinline__ float past_chunk(float a2, float sum, float h, float local) {
  const float f = fmaxf(__builtin_amdgcn_exp2f(0.5f * a2 * sum), 1.17549435e-38f);
  return fmaf(f * h, f, local);
}

// h through `n` summaries from index c0 (local alone where a prompt starts inside);
// put(c, h) sees the state before each.
template <class Put>
__device__ __forceinline__ float fold(const float* local, const float* sum_dt, size_t nd, int Di, size_t i, int d,
                                      float a2, int c0, int n, float h, float* total, Put put) {
  for (int q = 0; q < n; q += kCarryAhead) {
    float l[kCarryAhead], sd[kCarryAhead];
#pragma unroll
    for (int k = 0; k < kCarryAhead; ++k) {
      const int c = c0 + min(q + k, n - 1);
      l[k] = local[c * nd + i];
      sd[k] = sum_dt[static_cast<size_t>(c) * Di + d];
    }
#pragma unroll
    for (int k = 0; k < kCarryAhead; ++k) {
      if (q + k >= n) break;
      put(c0 + q + k, h);
      h = sd[k] < 0.f ? l[k] : past_chunk(a2, sd[k], h, l[k]);
      *total = sd[k] < 0.f || *total < 0.f ? -1.f : *total + sd[k];
    }
  }
  return h;
}

// The summary of each group of chunks (all but the last group's), a thread per state and group.
template <class E>
__global__ __launch_bounds__(256) void mixer_group_kernel(Mixer<E> g) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x, nd = static_cast<size_t>(g.N) * g.Di;
  if (i >= nd) return;
  const int n = static_cast<int>(i / g.Di), d = static_cast<int>(i % g.Di), q = static_cast<int>(blockIdx.y);
  const float a2 = -expf(g.a_log[static_cast<size_t>(d) * g.N + n]) * kLog2e;
  float total = 0.f;
  const float h = fold(g.local, g.sum_dt, nd, g.Di, i, d, a2, q * g.group, g.group, 0.f, &total, [](int, float) {});
  g.group_local[q * nd + i] = h;
  if (n == 0) g.group_dt[static_cast<size_t>(q) * g.Di + d] = total;
}

// carry[c], the state before chunk c: through the groups before, then the group's chunks.
template <class E>
__global__ __launch_bounds__(256) void mixer_carry_kernel(Mixer<E> g) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x, nd = static_cast<size_t>(g.N) * g.Di;
  if (i >= nd) return;
  const int n = static_cast<int>(i / g.Di), d = static_cast<int>(i % g.Di), q = static_cast<int>(blockIdx.y);
  const float a2 = -expf(g.a_log[static_cast<size_t>(d) * g.N + n]) * kLog2e;
  float total = 0.f;
  float h = fold(g.group_local, g.group_dt, nd, g.Di, i, d, a2, 0, q, 0.f, &total, [](int, float) {});
  const int c0 = q * g.group, n_own = min(g.group, g.n_chunks - c0);
  fold(g.local, g.sum_dt, nd, g.Di, i, d, a2, c0, n_own, h, &total, [&](int c, float v) { g.carry[c * nd + i] = v; });
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class E, int NB, int KT>
int launch_scan(const Mixer<E>& g, bool out, bool dt, int n_base, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((g.Di + kScanThreads - 1) / kScanThreads), static_cast<unsigned>(g.n_chunks));
  auto kern = out ? (dt ? mixer_scan_kernel<E, NB, KT, true, true> : mixer_scan_kernel<E, NB, KT, true, false>)
                  : (dt ? mixer_scan_kernel<E, NB, KT, false, true> : mixer_scan_kernel<E, NB, KT, false, false>);
  const bool vec = aligned16(g.dt_proj) && g.R % (16 / static_cast<int>(sizeof(E))) == 0;
  hipLaunchKernelGGL(kern, grid, dim3(kScanThreads), 0, st, g, n_base, vec);
  return launch_check("mixer_scan_kernel");
}

// One pass over all states, a block of them at a time; `dt`: the first block forms dt.
template <class E>
int launch_scans(const Mixer<E>& g, bool out, bool dt, hipStream_t st) {
  for (int n_base = 0; n_base < g.N; n_base += 32, dt = false) {
    const int left = g.N - n_base;
    const bool k4 = g.K <= 4;
    int rc;
    if (left <= 8) rc = k4 ? launch_scan<E, 8, 4>(g, out, dt, n_base, st) : launch_scan<E, 8, 8>(g, out, dt, n_base, st);
    else if (left <= 16) rc = k4 ? launch_scan<E, 16, 4>(g, out, dt, n_base, st) : launch_scan<E, 16, 8>(g, out, dt, n_base, st);
    else rc = k4 ? launch_scan<E, 32, 4>(g, out, dt, n_base, st) : launch_scan<E, 32, 8>(g, out, dt, n_base, st);
    if (rc) return rc;
  }
  return OSSM_OK;
}

template <class E>
bool vec8(const E* p, int row) { return aligned16(p) && row % (16 / static_cast<int>(sizeof(E))) == 0; }

// A stretch of the workspace of at least n floats whose end, the next one's start, is on 256
// bytes: vectors of 16 bytes are stored to it.
constexpr size_t stretch(size_t n) { return (n + 63) / 64 * 64; }
static_assert(stretch(18 * 299 * 83) % 4 == 0, "16-byte starts");

constexpr int kTokenRows = 2;  // rows of a workgroup of token_scan_kernel where there are many

template <class E>
int step(Mixer<E> g, StreamCall& call, hipStream_t st) {
  // Few rows: one each, in small workgroups, for the latency.  Many share the weights, the
  // projection's on the matrix cores where every row is whole vectors, from 400 channels a CU
  // on (a row at a time and shared, us of a step: 32 rows of d_inner 2048 15 and 16, 64 18.5 and
  // 17.4, 128 28 and 21; 128 of 512 13 and 14, 384 21 and 17), the scan's from 16 waves of
  // channels a CU on, what it holds at once (128 of 2048 21 and 24, 192 32 and 27).
  const int64_t channels = static_cast<int64_t>(g.rows) * g.Di, cus = std::max(1, device_cu_count(call.device()));
  const bool many = channels >= 400 * cus, many_scan = channels >= 16 * kWave * cus, k4 = g.K <= 4;
  const int e16 = 16 / static_cast<int>(sizeof(E));
  const bool tiles = many && g.Di % 8 == 0 && g.ld % e16 == 0 && aligned16(g.xz) && aligned16(g.conv_state) &&
                     aligned16(g.conv_w) && aligned16(g.conv_b) && aligned16(g.x_proj);
  g.n_blocks = (g.Di + (tiles ? kTileK : kProjBlock) - 1) / (tiles ? kTileK : kProjBlock);
  const int rows_per = tiles ? kTileRows : many ? 8 : 1;
  const int64_t groups = static_cast<int64_t>(g.n_blocks) * ((g.rows + rows_per - 1) / rows_per);
  if (int rc = check_grid("mixer_step", groups, tiles ? kTileThreads : kProjThreads)) return rc;
  const size_t part = stretch(static_cast<size_t>(g.n_blocks) * g.rows * g.Nc);
  void* ws = nullptr;
  if (int rc = acquire_workspace(call, (part + static_cast<size_t>(g.rows) * g.Di) * sizeof(float), &ws)) return rc;
  g.part = static_cast<float*>(ws);
  g.u = g.part + part;
  const bool vx = vec8(g.x_proj, g.Di);
  if (tiles) {
    hipLaunchKernelGGL(k4 ? (token_tile_kernel<E, 4>) : (token_tile_kernel<E, 8>), dim3(static_cast<unsigned>(groups)), dim3(kTileThreads), 0, st, g);
    if (int rc = launch_check("token_tile_kernel")) return rc;
  } else {
    auto proj = many ? (k4 ? token_proj_kernel<E, 8, 4> : token_proj_kernel<E, 8, 8>)
                     : (k4 ? token_proj_kernel<E, 1, 4> : token_proj_kernel<E, 1, 8>);
    hipLaunchKernelGGL(proj, dim3(static_cast<unsigned>(groups)), dim3(kProjThreads), 0, st, g, vx);
    if (int rc = launch_check("token_proj_kernel")) return rc;
  }
  const int rt = many_scan ? kTokenRows : 1, threads = many_scan ? 256 : 64;
  const dim3 gb(static_cast<unsigned>((g.Di + threads - 1) / threads), static_cast<unsigned>((g.rows + rt - 1) / rt));
  const int Rq = (g.R + 15) / 16 * 16, Nq = (g.N + 15) / 16 * 16;
  const size_t lds = static_cast<size_t>(rt) * (Rq + 2 * Nq) * sizeof(float);
  const bool vec = vec8(g.dt_proj, g.R) && vec8(g.a_log, g.N);
  hipLaunchKernelGGL(many_scan ? (vec ? token_scan_kernel<E, kTokenRows, true> : token_scan_kernel<E, kTokenRows, false>)
                          : (vec ? token_scan_kernel<E, 1, true> : token_scan_kernel<E, 1, false>),
                     gb, dim3(threads), lds, st, g, Rq, Nq);
  return launch_check("token_scan_kernel");
}

int64_t padded_states(int64_t n) { return n <= 8 ? 8 : n <= 16 ? 16 : (n + 31) / 32 * 32; }
int64_t padded_rank(int64_t r) { return (r + 15) / 16 * 16; }

// prompt_sum_kernel's workgroups: of the sums, and of the prompts it finishes.
int64_t prompt_sum_groups(int64_t rows, int64_t r, int64_t n) {
  return (rows * (padded_rank(r) + 2 * padded_states(n)) + 255) / 256;
}
int64_t prompt_finishers(int64_t di, int64_t n_seqs) { return (di + 255) / 256 * n_seqs; }

template <class E>
int prompt(Mixer<E> g, StreamCall& call, hipStream_t st) {
  const int64_t cus = std::max(1, device_cu_count(call.device()));
  // the channels split among enough workgroups for four a CU: up to 32 ways where a few
  // tiles of rows would leave the card empty, else eight (each adds its sums' traffic)
  const int64_t row_tiles = (g.rows + kPtRows - 1) / kPtRows, col_groups = (g.Nc + kPtCols - 1) / kPtCols;
  const int64_t k_steps = (g.Di + kPtK - 1) / kPtK;
  const int64_t ways = std::max<int64_t>(1, std::min<int64_t>({row_tiles * col_groups * 32 <= cus ? 32 : 8, k_steps, 4 * cus / std::max<int64_t>(1, row_tiles * col_groups)}));
  const int per_split = static_cast<int>((k_steps + ways - 1) / ways) * kPtK;
  g.n_blocks = (g.Di + per_split - 1) / per_split;
  g.Npad = static_cast<int>(padded_states(g.N));
  g.Rp = static_cast<int>(padded_rank(g.R));
  // enough chunks for four waves on each SIMD, of 16 tokens at least
  const int64_t waves = (g.Di + kWave - 1) / kWave;
  const int64_t want = std::max<int64_t>(1, 16 * cus / waves);
  g.chunk = static_cast<int>(std::max<int64_t>({16, (g.rows + want - 1) / want, (g.rows + 65534) / 65535}));
  g.n_chunks = (g.rows + g.chunk - 1) / g.chunk;
  // groups of about the square root of the chunks: as many steps through the groups as
  // through one's chunks
  g.group = 8;
  while (g.group * g.group < g.n_chunks) g.group += 8;
  g.n_groups = std::max(1, (g.n_chunks + g.group - 1) / g.group);
  const size_t nd = static_cast<size_t>(g.N) * g.Di;
  const bool carries = g.n_chunks > 1;
  size_t at = 0;
  const auto take = [&](size_t n) { const size_t o = at; at += stretch(n); return o; };
  const size_t o_part = take(static_cast<size_t>(g.n_blocks) * g.rows * g.Nc);
  const size_t o_planes = take((3 * static_cast<size_t>(g.rows) * g.Rp + 1) / 2);
  const size_t o_bc = take(static_cast<size_t>(g.rows) * 2 * g.Npad);
  const bool keep_dt = carries || g.N > 32;  // a pass reads what an earlier one formed
  const size_t o_dt = take(keep_dt ? static_cast<size_t>(g.rows) * g.Di : 0);
  const size_t o_local = take(carries ? g.n_chunks * nd : 0);
  const size_t o_carry = take(carries ? g.n_chunks * nd : 0);
  const size_t o_sum = take(carries ? static_cast<size_t>(g.n_chunks) * g.Di : 0);
  const size_t o_glocal = take(carries ? g.n_groups * nd : 0);
  const size_t o_gsum = take(carries ? static_cast<size_t>(g.n_groups) * g.Di : 0);
  const size_t o_init = take(g.resume != nullptr ? g.n_seqs * nd : 0);
  const size_t o_y = take(g.N > 32 ? static_cast<size_t>(g.rows) * g.Di : 0);
  void* ws = nullptr;
  if (int rc = acquire_workspace(call, at * sizeof(float), &ws)) return rc;
  float* f = static_cast<float*>(ws);
  g.part = f + o_part;
  g.planes = reinterpret_cast<uint16_t*>(f + o_planes);
  g.bc = f + o_bc;
  g.dt = keep_dt ? f + o_dt : nullptr;
  g.local = f + o_local;
  g.carry = f + o_carry;
  g.sum_dt = f + o_sum;
  g.group_local = f + o_glocal;
  g.group_dt = f + o_gsum;
  g.y_sum = f + o_y;
  if (g.rows > 0) {
    const bool k4 = g.K <= 4;
    // quads of channels in one load each
    const bool quads = g.Di % 4 == 0 && g.ld % 4 == 0 && aligned16(g.xz) && aligned16(g.conv_w);
    hipLaunchKernelGGL(quads ? (k4 ? prompt_proj_kernel<E, 4, true> : prompt_proj_kernel<E, 8, true>)
                             : (k4 ? prompt_proj_kernel<E, 4, false> : prompt_proj_kernel<E, 8, false>),
                       dim3(static_cast<unsigned>(row_tiles * g.n_blocks * col_groups)), dim3(256), 0, st, g, per_split,
                       vec8(g.x_proj, g.Di));
    if (int rc = launch_check("prompt_proj_kernel")) return rc;
    const unsigned sum_groups = static_cast<unsigned>(prompt_sum_groups(g.rows, g.R, g.N));
    const unsigned finishers = g.resume == nullptr ? static_cast<unsigned>(prompt_finishers(g.Di, g.n_seqs)) : 0;
    hipLaunchKernelGGL(prompt_sum_kernel<E>, dim3(sum_groups + finishers), dim3(256), 0, st, g, sum_groups);
    if (int rc = launch_check("prompt_sum_kernel")) return rc;
    if (g.resume != nullptr) {
      g.init = f + o_init;
      hipLaunchKernelGGL(mixer_gather_kernel<E>, dim3(static_cast<unsigned>(std::min<size_t>(64, (nd + 255) / 256)),
                                                      static_cast<unsigned>(g.n_seqs)), dim3(256), 0, st, g);
      if (int rc = launch_check("mixer_gather_kernel")) return rc;
    }
    // dt in the first scan saves a launch where there are few waves (one prompt of 117
    // tokens at d_inner 2048 55 -> 49 us), and costs the scan its occupancy where there
    // are many (16384 tokens 456 -> 478, 25600 at d_inner 128 122 -> 126)
    const bool dt_in_scan = !carries || g.n_chunks * waves <= 4 * cus;
    if (!dt_in_scan) {
      const dim3 grid(static_cast<unsigned>((g.rows + kDtRows - 1) / kDtRows), static_cast<unsigned>((g.Di + kDtCols - 1) / kDtCols));
      hipLaunchKernelGGL(prompt_dt_kernel<E>, grid, dim3(256), 0, st, g,
                         aligned16(g.dt_proj) && g.R % (16 / static_cast<int>(sizeof(E))) == 0);
      if (int rc = launch_check("prompt_dt_kernel")) return rc;
    }
    if (carries) {
      if (int rc = launch_scans(g, false, dt_in_scan, st)) return rc;
      const unsigned nb = static_cast<unsigned>((nd + 255) / 256);
      if (g.n_groups > 1) {
        hipLaunchKernelGGL(mixer_group_kernel<E>, dim3(nb, static_cast<unsigned>(g.n_groups - 1)), dim3(256), 0, st, g);
        if (int rc = launch_check("mixer_group_kernel")) return rc;
      }
      hipLaunchKernelGGL(mixer_carry_kernel<E>, dim3(nb, static_cast<unsigned>(g.n_groups)), dim3(256), 0, st, g);
      if (int rc = launch_check("mixer_carry_kernel")) return rc;
    }
    if (int rc = launch_scans(g, true, !carries, st)) return rc;
    if (g.resume == nullptr) return OSSM_OK;  // the sums' launch has finished the prompts
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
      ((rows + 7) / 8) * ((di + 127) / 128) > INT_MAX / 2 || ((rows + 63) / 64) * 8 * ((r + 2 * n + 127) / 128) > INT_MAX)
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
  if (int rc = check_grid("mixer_prompt", prompt_sum_groups(rows, dt_rank, d_state) + prompt_finishers(d_inner, n_seqs), 256))
    return rc;
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
