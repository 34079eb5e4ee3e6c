// Layer norm of rows, alone or of a residual sum, forward and backward
// (ossm_layer_norm_forward, ossm_layer_norm_backward):
//
//   s = x + residual, rounded to its type;  c = s - mean(s);  rstd = (mean(c^2) + eps)^-1/2
//   y = c rstd w + b
//   g = gy w;  ds = rstd (g - mean(g) - n mean(g n)) + gs,  n = c rstd
//   dw = sum over rows of gy n,  db = sum over rows of gy
//
// All of it is bound by memory: [32768, 2048] in bf16 with a residual takes 92 to 103 us forward (5.2
// to 5.8 TB/s) and 103 to 117 backward (4.6 to 5.2), a copy runs at 4.9; short calls by their
// latency, 4 us at [4, 2048].  A group of G lanes holds a whole row in registers, in
// vectors of 16 bytes, so that every tensor is read once and the squares are summed about
// the mean (sums of the elements' own squares would lose what a large mean takes).  G is the
// least that holds the row: 8 to 64 lanes share a wave with other rows and need no
// barrier, longer rows take a workgroup.  The groups walk the rows with the weights kept in
// registers; in the backward each keeps its share of dw and db there too, workgroups
// leave theirs as partial sums, and a second kernel adds those in a fixed order: results
// are bitwise repeatable.

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <string>

#include "../../include/ossm_lm.h"
#include "lm_types.hpp"
#include "lm_vector.hpp"
#include "runtime.hpp"

namespace ossm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxThreads = 1024;

template <class E>
constexpr int kVec = 16 / static_cast<int>(sizeof(E));

template <class E, class WT>
struct Norm {
  const E* x;
  const E* residual;
  const WT* weight;
  const WT* bias;
  E* y;
  E* sum;
  float* mean;
  float* rstd;
  const E* gy;
  const E* gs;
  E* gx;
  float* partial;  // [workgroups, 2, D]
  long long ld_x, ld_res, ld_gy, ld_gs, rows;
  float eps;
  int D;
};

// Threads of a workgroup whose rows take G lanes each.
template <int G>
constexpr int kBlockOf = G > 64 ? G : kThreads;

// Two sums over a row's lanes at once.
template <int G>
__device__ __forceinline__ float2 row_sums(float a, float b, float2* s_sum) {
  constexpr int L = G < 64 ? G : 64;
  a = lanes_sum<L>(a);
  b = lanes_sum<L>(b);
  if constexpr (G > 64) {
    __syncthreads();  // the previous sums are read
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x / 64] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) {
      a += s_sum[w].x;
      b += s_sum[w].y;
    }
  }
  return make_float2(a, b);
}

template <class WT, int NV, int W, int G>
__device__ __forceinline__ void load_weights(const WT* p, int D, int lane, float none, float (&w)[NV][W]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * G + lane) * W;
    Vec<WT, W> t;
    t.zero();
    if (p != nullptr && at < D) t.load(p + at, D - at);
#pragma unroll
    for (int k = 0; k < W; ++k) w[j][k] = p != nullptr ? t.get(k) : none;
  }
}

// The mean is the row's first element, the pivot, and the mean of the differences from it: in a row far
// from zero, whose elements differ little, those are exact, and zero where all are equal.  (A mean of
// the elements' own sum is off by many roundings of its size, which every deviation would carry: its square
// could pass the variance and eps, NaN at equal elements of 2e8.)  The mean is still rounded to its own
// size, by no more than the elements differ, which the deviations all carry: their own mean, `rest`, is
// taken off again.
struct Row {
  float rest, rstd;
};
__device__ __forceinline__ Row row_of(float2 sums, float inv, float eps) {
  const float rest = sums.y * inv;
  return {rest, 1.f / sqrtf(fmaf(-rest, rest, sums.x * inv) + eps)};
}

// The first element of row r, of the sum where there is a residual.
template <class E, class WT>
__device__ __forceinline__ float pivot_of(const Norm<E, WT>& g, E x, E residual) {
  return g.residual != nullptr ? to_f(from_f<E>(to_f(x) + to_f(residual))) : to_f(x);
}

// a b, rounded: the mean of gy w is taken off the same numbers that it is of.  Fused into the
// difference, the product's rounding would stay behind, times rstd, which in a row of (nearly)
// equal elements is eps^-1/2.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// RAGGED: D is no multiple of a vector, and rows share lines.
template <class E, class WT, int G, int NV, bool RAGGED>
__global__ __launch_bounds__(kBlockOf<G>) void norm_forward_kernel(Norm<E, WT> g) {
  constexpr int W = kVec<E>, kRows = kBlockOf<G> / G;
  __shared__ float2 s_sum[G > 64 ? G / 64 : 1];
  const int lane = threadIdx.x % G;
  const auto left_of = [&](int at) { return RAGGED ? g.D - at : W; };  // a vector's elements in the row
  const float inv = 1.f / static_cast<float>(g.D);
  float w[NV][W], b[NV][W];
  load_weights<WT, NV, W, G>(g.weight, g.D, lane, 1.f, w);
  load_weights<WT, NV, W, G>(g.bias, g.D, lane, 0.f, b);
  const long long step = static_cast<long long>(gridDim.x) * kRows;
  long long r = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / G;
  Vec<E, W> raw[NV], res[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) raw[j].zero(), res[j].zero();
  E first{}, res_first{};
  const auto fetch = [&](long long row) {
    if (row >= g.rows) return;
    if constexpr (G >= 64) {  // fewer lanes hand on the first one's
      first = g.x[row * g.ld_x];
      if (g.residual != nullptr) res_first = g.residual[row * g.ld_res];
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * G + lane) * W;
      if (at < g.D) raw[j].load(g.x + row * g.ld_x + at, left_of(at), RAGGED ? (g.rows - 1 - row) * g.ld_x + g.D - at : 0);
      if (at < g.D && g.residual != nullptr)
        res[j].load(g.residual + row * g.ld_res + at, left_of(at), RAGGED ? (g.rows - 1 - row) * g.ld_res + g.D - at : 0);
    }
  };
  fetch(r);
  for (; r < g.rows; r += step) {
    float v[NV][W], total = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * G + lane) * W;
      if (RAGGED && at < g.D) {
        raw[j].keep(g.D - at);
        res[j].keep(g.D - at);
      }
      if (at < g.D && g.residual != nullptr) {
        float t[W];
#pragma unroll
        for (int k = 0; k < W; ++k) t[k] = raw[j].get(k) + res[j].get(k);
        raw[j].set(t);
        raw[j].template store<!RAGGED>(g.sum + r * g.D + at, left_of(at));
      }
    }
    float pivot;
    if constexpr (G >= 64) pivot = pivot_of(g, first, res_first);
    else pivot = __shfl(raw[0].get(0), 0, G);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * G + lane) * W;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        v[j][k] = raw[j].get(k);
        total += at + k < g.D ? v[j][k] - pivot : 0.f;
      }
    }
    fetch(r + step);  // the next row comes in while this one is summed
    __builtin_amdgcn_sched_barrier(0);
    const float mean = pivot + row_sums<G>(total, 0.f, s_sum).x / static_cast<float>(g.D);
    float square = 0.f, rest = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        v[j][k] = (j * G + lane) * W + k < g.D ? v[j][k] - mean : 0.f;
        square = fmaf(v[j][k], v[j][k], square);
        rest += v[j][k];
      }
    const Row row = row_of(row_sums<G>(square, rest, s_sum), inv, g.eps);
    if (lane == 0 && g.mean != nullptr) {
      g.mean[r] = mean + row.rest;
      g.rstd[r] = row.rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * G + lane) * W;
      float t[W];
      Vec<E, W> out;
#pragma unroll
      for (int k = 0; k < W; ++k) t[k] = fmaf((v[j][k] - row.rest) * row.rstd, w[j][k], b[j][k]);
      out.set(t);
      if (at < g.D) out.template store<!RAGGED>(g.y + r * g.D + at, left_of(at));
    }
  }
}

template <class E, class WT, int G, int NV, bool RAGGED>
__global__ __launch_bounds__(kBlockOf<G>) void norm_backward_kernel(Norm<E, WT> g) {
  constexpr int W = kVec<E>, kRows = kBlockOf<G> / G;
  __shared__ float2 s_sum[G > 64 ? G / 64 : 1];
  __shared__ float s_part[G <= 64 ? 2 : 1][G <= 64 ? G * NV * W : 1];
  const int lane = threadIdx.x % G;
  const auto left_of = [&](int at) { return RAGGED ? g.D - at : W; };  // a vector's elements in the row
  const float inv = 1.f / static_cast<float>(g.D);
  float w[NV][W], dw[NV][W], db[NV][W];
  load_weights<WT, NV, W, G>(g.weight, g.D, lane, 1.f, w);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < W; ++k) dw[j][k] = db[j][k] = 0.f;
  const long long step = static_cast<long long>(gridDim.x) * kRows;
  long long r = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / G;
  Vec<E, W> s_in[NV], gy_in[NV], gs_in[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) s_in[j].zero(), gy_in[j].zero(), gs_in[j].zero();
  float mean_in = 0.f, rstd_in = 0.f;
  const auto fetch = [&](long long row) {
    if (row >= g.rows) return;
    mean_in = g.mean[row];
    rstd_in = g.rstd[row];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * G + lane) * W;
      if (at < g.D) {
        const long long left = g.rows - 1 - row;
        s_in[j].load(g.x + row * g.ld_x + at, left_of(at), RAGGED ? left * g.ld_x + g.D - at : 0);
        gy_in[j].load(g.gy + row * g.ld_gy + at, left_of(at), RAGGED ? left * g.ld_gy + g.D - at : 0);
        if (g.gs != nullptr) gs_in[j].load(g.gs + row * g.ld_gs + at, left_of(at), RAGGED ? left * g.ld_gs + g.D - at : 0);
      }
    }
  };
  constexpr bool kAhead = NV * W <= 8;  // where there are registers for a second row
  if (kAhead) fetch(r);
  for (; r < g.rows; r += step) {
    if (!kAhead) fetch(r);
    const float rstd = rstd_in, mean = mean_in;
    Vec<E, W> s[NV], gy[NV], gs[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      s[j] = s_in[j], gy[j] = gy_in[j], gs[j] = gs_in[j];
      const int at = (j * G + lane) * W;
      if (RAGGED && at < g.D) {
        s[j].keep(g.D - at);
        gy[j].keep(g.D - at);
      }
    }
    if (kAhead) {
      fetch(r + step);  // the next row comes in while this one is summed
      __builtin_amdgcn_sched_barrier(0);
    }
    float m1 = 0.f, m2 = 0.f;  // past the row's end gy is zero
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float n = (s[j].get(k) - mean) * rstd, o = gy[j].get(k), q = product(o, w[j][k]);
        dw[j][k] = fmaf(o, n, dw[j][k]);
        db[j][k] += o;
        m1 += q;
        m2 = fmaf(q, n, m2);
      }
    const float2 m = row_sums<G>(m1, m2, s_sum);
    m1 = m.x * inv;
    m2 = m.y * inv;
    // n and gy w are formed again from the packed row: kept, they would take four times its registers
#pragma unroll
    for (int j = 0; j < NV && kAhead; ++j)
#pragma unroll
      for (int i = 0; i < Vec<E, W>::kWords; ++i) asm volatile("" : "+v"(s[j].w[i]), "+v"(gy[j].w[i]));
    if (g.gx != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * G + lane) * W;
        if (at >= g.D) continue;
        float t[W];
        Vec<E, W> out;
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const float n = (s[j].get(k) - mean) * rstd;
          t[k] = fmaf(rstd, fmaf(-n, m2, product(gy[j].get(k), w[j][k]) - m1), gs[j].get(k));  // no gs: zeros
        }
        out.set(t);
        out.template store<!RAGGED>(g.gx + r * g.D + at, left_of(at));
      }
    }
  }
  if (g.partial == nullptr) return;
  float* part = g.partial + static_cast<size_t>(blockIdx.x) * 2 * g.D;
  if constexpr (G <= 64) {
    // the groups of a wave by their lanes, the waves one after another
#pragma unroll
    for (int o = 32; o >= G; o >>= 1)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < W; ++k) {
          dw[j][k] += __shfl_xor(dw[j][k], o);
          db[j][k] += __shfl_xor(db[j][k], o);
        }
    for (int v = 0; v < kThreads / 64; ++v) {
      if (static_cast<int>(threadIdx.x) / 64 == v && (threadIdx.x & 63) < G) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int k = 0; k < W; ++k) {
            const int at = (j * G + lane) * W + k;
            s_part[0][at] = v == 0 ? dw[j][k] : s_part[0][at] + dw[j][k];
            s_part[1][at] = v == 0 ? db[j][k] : s_part[1][at] + db[j][k];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < g.D; i += kThreads) {
      part[i] = s_part[0][i];
      part[g.D + i] = s_part[1][i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * G + lane) * W;
      if (at >= g.D) continue;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if (at + k >= g.D) break;
        part[at + k] = dw[j][k];
        part[g.D + at + k] = db[j][k];
      }
    }
  }
}

// Rows longer than a workgroup's registers hold: the same sums in passes over the row, from
// the caches after the first.  f(first element, its elements, vectors of each tensor).
template <class E, int N, class F>
__device__ __forceinline__ void each_vector(const E* const (&rows)[N], int D, F f) {
  constexpr int W = kVec<E>;
  for (int at = static_cast<int>(threadIdx.x) * W; at < D; at += kMaxThreads * W) {
    Vec<E, W> v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i].zero();
      if (rows[i] != nullptr) v[i].load(rows[i] + at, D - at);
    }
    f(at, min(W, D - at), v);
  }
}

template <class E, class WT>
__global__ __launch_bounds__(kMaxThreads) void long_forward_kernel(Norm<E, WT> g) {
  constexpr int W = kVec<E>;
  __shared__ float2 s_sum[kMaxThreads / 64];
  const float inv = 1.f / static_cast<float>(g.D);
  for (long long r = blockIdx.x; r < g.rows; r += gridDim.x) {
    const E* in[1] = {g.x + r * g.ld_x};
    const float pivot = pivot_of(g, *in[0], g.residual != nullptr ? g.residual[r * g.ld_res] : E{});
    float total = 0.f;
    if (g.residual != nullptr) {
      const E* const both[2] = {in[0], g.residual + r * g.ld_res};
      each_vector(both, g.D, [&](int at, int n, Vec<E, W>(&v)[2]) {
        float t[W];
#pragma unroll
        for (int k = 0; k < W; ++k) t[k] = v[0].get(k) + v[1].get(k);
        v[0].set(t);
#pragma unroll
        for (int k = 0; k < W; ++k) total += k < n ? v[0].get(k) - pivot : 0.f;
        v[0].template store<false>(g.sum + r * g.D + at, n);
      });
      in[0] = g.sum + r * g.D;  // a thread reads back its own elements
    } else {
      each_vector(in, g.D, [&](int, int n, Vec<E, W>(&v)[1]) {
#pragma unroll
        for (int k = 0; k < W; ++k) total += k < n ? v[0].get(k) - pivot : 0.f;
      });
    }
    const float mean = pivot + row_sums<kMaxThreads>(total, 0.f, s_sum).x / static_cast<float>(g.D);
    float square = 0.f, rest = 0.f;
    each_vector(in, g.D, [&](int, int n, Vec<E, W>(&v)[1]) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float c = k < n ? v[0].get(k) - mean : 0.f;
        square = fmaf(c, c, square);
        rest += c;
      }
    });
    const Row row = row_of(row_sums<kMaxThreads>(square, rest, s_sum), inv, g.eps);
    if (threadIdx.x == 0 && g.mean != nullptr) {
      g.mean[r] = mean + row.rest;
      g.rstd[r] = row.rstd;
    }
    each_vector(in, g.D, [&](int at, int n, Vec<E, W>(&v)[1]) {
      float w[1][W], b[1][W], t[W];
      load_weights<WT, 1, W, kMaxThreads>(g.weight, g.D, at / W, 1.f, w);
      load_weights<WT, 1, W, kMaxThreads>(g.bias, g.D, at / W, 0.f, b);
#pragma unroll
      for (int k = 0; k < W; ++k) t[k] = fmaf((v[0].get(k) - mean - row.rest) * row.rstd, w[0][k], b[0][k]);
      v[0].set(t);
      v[0].template store<false>(g.y + r * g.D + at, n);
    });
  }
}

template <class E, class WT>
__global__ __launch_bounds__(kMaxThreads) void long_backward_kernel(Norm<E, WT> g) {
  constexpr int W = kVec<E>;
  __shared__ float2 s_sum[kMaxThreads / 64];
  const float inv = 1.f / static_cast<float>(g.D);
  for (long long r = blockIdx.x; r < g.rows; r += gridDim.x) {
    const E* const in[3] = {g.x + r * g.ld_x, g.gy + r * g.ld_gy, g.gs != nullptr ? g.gs + r * g.ld_gs : nullptr};
    const E* const two[2] = {in[0], in[1]};
    const float mean = g.mean[r], rstd = g.rstd[r];
    float m1 = 0.f, m2 = 0.f;
    each_vector(two, g.D, [&](int at, int, Vec<E, W>(&v)[2]) {
      float w[1][W];
      load_weights<WT, 1, W, kMaxThreads>(g.weight, g.D, at / W, 1.f, w);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float q = product(v[1].get(k), w[0][k]);
        m1 += q;
        m2 = fmaf(q, (v[0].get(k) - mean) * rstd, m2);
      }
    });
    const float2 m = row_sums<kMaxThreads>(m1, m2, s_sum);
    m1 = m.x * inv;
    m2 = m.y * inv;
    each_vector(in, g.D, [&](int at, int n, Vec<E, W>(&v)[3]) {
      float w[1][W], t[W];
      load_weights<WT, 1, W, kMaxThreads>(g.weight, g.D, at / W, 1.f, w);
#pragma unroll
      for (int k = 0; k < W; ++k)
        t[k] = fmaf(rstd, fmaf(-(v[0].get(k) - mean) * rstd, m2, product(v[1].get(k), w[0][k]) - m1), v[2].get(k));
      v[0].set(t);
      v[0].template store<false>(g.gx + r * g.D + at, n);
    });
  }
}

// dw and db of such rows: every n_parts-th row for the vectors of a workgroup's threads.
template <class E, class WT>
__global__ __launch_bounds__(kThreads) void long_columns_kernel(Norm<E, WT> g, int n_parts, int n_cols) {
  constexpr int W = kVec<E>;
  const int part = static_cast<int>(blockIdx.x) / n_cols, at = (static_cast<int>(blockIdx.x) % n_cols * kThreads + threadIdx.x) * W;
  if (at >= g.D) return;
  float dw[W] = {}, db[W] = {};
  for (long long r = part; r < g.rows; r += n_parts) {
    Vec<E, W> s, gy;
    s.load(g.x + r * g.ld_x + at, g.D - at);
    gy.load(g.gy + r * g.ld_gy + at, g.D - at);
    const float mean = g.mean[r], rstd = g.rstd[r];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      dw[k] = fmaf(gy.get(k), (s.get(k) - mean) * rstd, dw[k]);
      db[k] += gy.get(k);
    }
  }
  float* out = g.partial + static_cast<size_t>(part) * 2 * g.D;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if (at + k >= g.D) break;
    out[at + k] = dw[k];
    out[g.D + at + k] = db[k];
  }
}

// dw and db from n partial sums.
template <class WT>
__global__ __launch_bounds__(kSumThreads) void norm_sum_kernel(const float* partial, int n, int D, WT* dw, WT* db) {
  const long long cols = 2ll * D, i = static_cast<long long>(blockIdx.x) * kSumColumns + threadIdx.x;
  const double t = column_sum(partial, n, cols, cols);
  if (threadIdx.x >= kSumColumns || i >= cols) return;
  WT* out = i < D ? dw : db;
  if (out != nullptr) out[i < D ? i : i - D] = from_f<WT>(static_cast<float>(t));
}

// Calls f(G, NV) with the least group of lanes that holds D elements in up to MAXV vectors each
// where there are lanes enough (or more of 1024 lanes), or returns false.
template <class E, int MAXV, class F>
bool with_group(int64_t D, F f) {
  constexpr int W = kVec<E>;
  using std::integral_constant;
#define OSSM_GROUP(G, NV) \
  if (D <= int64_t(G) * (NV) * W) return f(integral_constant<int, G>{}, integral_constant<int, NV>{}), true
  OSSM_GROUP(8, 1);
  OSSM_GROUP(16, 1);
  OSSM_GROUP(32, 1);
  OSSM_GROUP(64, 1);
  if constexpr (MAXV > 1) {
    OSSM_GROUP(64, 2);
    OSSM_GROUP(128, 2);
    OSSM_GROUP(256, 2);
    OSSM_GROUP(512, 2);
  } else {
    OSSM_GROUP(128, 1);
    OSSM_GROUP(256, 1);
    OSSM_GROUP(512, 1);
    OSSM_GROUP(1024, 1);
  }
  if constexpr (sizeof(E) == 4) OSSM_GROUP(1024, 2);
  if constexpr (MAXV > 1) OSSM_GROUP(1024, 16 / W);
#undef OSSM_GROUP
  return false;
}

// The forward takes two vectors a lane, the backward, whose sums take twice the registers, one:
// forward and backward of [32768, 2048] in bf16 with a residual at one vector 98 and 115 us, at
// two 91 and 131, at four 93 and 138.
constexpr int kForwardVecs = 2, kBackwardVecs = 1;
constexpr int kForwardWaves = 32, kBackwardWaves = 16;  // a CU

// Workgroups that walk the rows: as many as the card holds at once.
int64_t walkers(int64_t rows, int rows_each, int threads, int cus, int waves) {
  const int64_t most = int64_t(cus > 0 ? cus : 256) * (waves * 64 / threads > 0 ? waves * 64 / threads : 1);
  const int64_t need = (rows + rows_each - 1) / rows_each;
  return need < most ? need : most;
}

// In the backward each leaves two rows of partial sums too: at least four rows each, where
// that still leaves one for every CU.
int64_t summing_walkers(int64_t rows, int rows_each, int threads, int cus) {
  const int64_t need = (rows + rows_each - 1) / rows_each, few = need < cus ? need : cus;
  const int64_t most = walkers(rows, rows_each, threads, cus, kBackwardWaves);
  const int64_t want = need / 4 > few ? need / 4 : few;
  return want < most ? want : most;
}

template <class E, class WT>
int forward(Norm<E, WT> g, int cus, hipStream_t st) {
  const bool held = with_group<E, kForwardVecs>(g.D, [&](auto G, auto NV) {
    constexpr int kG = decltype(G)::value, kNV = decltype(NV)::value, kB = kBlockOf<kG>;
    const auto kern = g.D % kVec<E> != 0 ? norm_forward_kernel<E, WT, kG, kNV, true> : norm_forward_kernel<E, WT, kG, kNV, false>;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(walkers(g.rows, kB / kG, kB, cus, kForwardWaves))), dim3(kB), 0, st, g);
  });
  if (!held)
    hipLaunchKernelGGL((long_forward_kernel<E, WT>),
                       dim3(static_cast<unsigned>(walkers(g.rows, 1, kMaxThreads, cus, kForwardWaves))), dim3(kMaxThreads), 0,
                       st, g);
  return launch_check("norm_forward_kernel");
}

template <class E, class WT>
int backward(Norm<E, WT> g, WT* dw, WT* db, StreamCall& call, int cus) {
  hipStream_t st = call.stream();
  int64_t parts = 0;
  const bool held = with_group<E, kBackwardVecs>(g.D, [&](auto G, auto) {
    constexpr int kG = decltype(G)::value, kB = kBlockOf<kG>;
    parts = summing_walkers(g.rows, kB / kG, kB, cus > 0 ? cus : 256);
  });
  const int n_cols = (g.D + kThreads * kVec<E> - 1) / (kThreads * kVec<E>);
  if (!held) parts = walkers(g.rows, 16, kThreads, cus, 16 / (n_cols < 16 ? n_cols : 16));
  const bool sums = dw != nullptr || db != nullptr;
  if (sums) {
    void* p = nullptr;
    if (int rc = acquire_workspace(call, static_cast<size_t>(parts) * 2 * g.D * sizeof(float), &p)) return rc;
    g.partial = static_cast<float*>(p);
  }
  with_group<E, kBackwardVecs>(g.D, [&](auto G, auto NV) {
    constexpr int kG = decltype(G)::value, kNV = decltype(NV)::value, kB = kBlockOf<kG>;
    const auto kern = g.D % kVec<E> != 0 ? norm_backward_kernel<E, WT, kG, kNV, true> : norm_backward_kernel<E, WT, kG, kNV, false>;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(parts)), dim3(kB), 0, st, g);
  });
  if (!held) {
    if (g.gx != nullptr)
      hipLaunchKernelGGL((long_backward_kernel<E, WT>),
                         dim3(static_cast<unsigned>(walkers(g.rows, 1, kMaxThreads, cus, kForwardWaves))), dim3(kMaxThreads),
                         0, st, g);
    if (sums) {
      if (int rc = check_grid("layer_norm_backward", parts * n_cols, kThreads)) return rc;
      hipLaunchKernelGGL((long_columns_kernel<E, WT>), dim3(static_cast<unsigned>(parts * n_cols)), dim3(kThreads), 0, st, g,
                         static_cast<int>(parts), n_cols);
    }
  }
  if (int rc = launch_check("norm_backward_kernel")) return rc;
  if (!sums) return OSSM_OK;
  hipLaunchKernelGGL(norm_sum_kernel<WT>, dim3(static_cast<unsigned>((2ll * g.D + kSumColumns - 1) / kSumColumns)),
                     dim3(kSumThreads), 0, st,
                     g.partial, static_cast<int>(parts), g.D, dw, db);
  return launch_check("norm_sum_kernel");
}

int check_types(const char* what, int dtype, int wdtype, int64_t rows, int64_t dim) {
  if ((dtype != OSSM_F32 && dtype != OSSM_BF16) || (wdtype != OSSM_F32 && wdtype != dtype))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": unknown dtype");
  if (rows < 0 || dim < 0) return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  if (dim > INT_MAX / 16) return set_error(OSSM_ERR_UNSUPPORTED, std::string(what) + ": size exceeds launch limits");
  return OSSM_OK;
}

}  // namespace
}  // namespace ossm

using namespace ossm;

extern "C" {

int ossm_layer_norm_forward(int dtype, int weight_dtype, const void* x, int64_t ld_x, const void* residual,
                            int64_t ld_residual, const void* weight, const void* bias, float eps, void* y, void* sum,
                            float* mean, float* rstd, int64_t rows, int64_t dim, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "layer_norm_forward";
  if (int rc = check_types(what, dtype, weight_dtype, rows, dim)) return rc;
  if (rows == 0 || dim == 0) return OSSM_OK;
  if (!x || !y || (residual != nullptr) != (sum != nullptr) || (mean != nullptr) != (rstd != nullptr))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": null pointer");
  if (rows > 1 && (ld_x < dim || (residual && ld_residual < dim)))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": row stride below the row");
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  int dev = 0;
  if (int rc = hip_check(hipGetDevice(&dev), "hipGetDevice")) return rc;
  const int cus = device_cu_count(dev);
  const auto go = [&](auto e, auto w) {
    using E = decltype(e);
    using WT = decltype(w);
    Norm<E, WT> g{};
    g.x = static_cast<const E*>(x), g.ld_x = ld_x;
    g.residual = static_cast<const E*>(residual), g.ld_res = ld_residual;
    g.weight = static_cast<const WT*>(weight), g.bias = static_cast<const WT*>(bias);
    g.y = static_cast<E*>(y), g.sum = static_cast<E*>(sum), g.mean = mean, g.rstd = rstd;
    g.rows = rows, g.D = static_cast<int>(dim), g.eps = eps;
    return forward(g, cus, st);
  };
  if (dtype == OSSM_F32) return go(0.f, 0.f);
  return weight_dtype == OSSM_F32 ? go(bf16_t{}, 0.f) : go(bf16_t{}, bf16_t{});
}

int ossm_layer_norm_backward(int dtype, int weight_dtype, const void* grad_y, int64_t ld_grad_y, const void* grad_sum,
                             int64_t ld_grad_sum, const void* s, int64_t ld_s, const void* weight, const float* mean,
                             const float* rstd, void* grad_x, void* grad_weight, void* grad_bias, int64_t rows, int64_t dim,
                             ossm_stream_t stream_v) {
  clear_error();
  const char* what = "layer_norm_backward";
  if (int rc = check_types(what, dtype, weight_dtype, rows, dim)) return rc;
  if (rows == 0 || dim == 0) return OSSM_OK;
  if (int rc = check_grid(what, (2 * dim + kSumColumns - 1) / kSumColumns, kSumThreads)) return rc;
  if (!grad_y || !s || !mean || !rstd) return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": null pointer");
  if (rows > 1 && (ld_s < dim || ld_grad_y < dim || (grad_sum && ld_grad_sum < dim)))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": row stride below the row");
  StreamCall call(static_cast<hipStream_t>(stream_v));
  if (call.status()) return call.status();
  const int cus = device_cu_count(call.device());
  const auto go = [&](auto e, auto w) {
    using E = decltype(e);
    using WT = decltype(w);
    Norm<E, WT> g{};
    g.x = static_cast<const E*>(s), g.ld_x = ld_s;
    g.gy = static_cast<const E*>(grad_y), g.ld_gy = ld_grad_y;
    g.gs = static_cast<const E*>(grad_sum), g.ld_gs = ld_grad_sum;
    g.weight = static_cast<const WT*>(weight);
    g.mean = const_cast<float*>(mean), g.rstd = const_cast<float*>(rstd);
    g.gx = static_cast<E*>(grad_x);
    g.rows = rows, g.D = static_cast<int>(dim);
    return backward(g, static_cast<WT*>(grad_weight), static_cast<WT*>(grad_bias), call, cus);
  };
  if (dtype == OSSM_F32) return go(0.f, 0.f);
  return weight_dtype == OSSM_F32 ? go(bf16_t{}, 0.f) : go(bf16_t{}, bf16_t{});
}

}  // extern "C"
