// Layer norm of rows, alone or of a residual sum, forward and backward
// (ossm_layer_norm_forward, ossm_layer_norm_backward):
//
//   s = x + residual, rounded to its type;  c = s - mean(s);  rstd = (mean(c^2) + eps)^-1/2
//   y = c rstd w + b
//   g = gy w;  ds = rstd (g - mean(g) - n mean(g n)) + gs,  n = c rstd
//   dw = sum over rows of gy n,  db = sum over rows of gy
//
// All of it is bound by memory.  A group of G lanes holds a whole row in registers, in
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
constexpr int kBlockOf = G > kThreads ? G : kThreads;

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
    WT t[W];
    if (p != nullptr && at < D) load_part(p + at, D - at, t);
#pragma unroll
    for (int k = 0; k < W; ++k) w[j][k] = p != nullptr && at < D ? to_f(t[k]) : none;
  }
}

// A row's mean is rounded to its own size, which the deviations of a row far from zero
// would all carry: their own mean, `rest`, is taken off again.
struct Row {
  float rest, rstd;
};
__device__ __forceinline__ Row row_of(float2 sums, float inv, float eps) {
  const float rest = sums.y * inv;
  return {rest, 1.f / sqrtf(fmaf(-rest, rest, sums.x * inv) + eps)};
}

template <class E, class WT, int G, int NV>
__global__ __launch_bounds__(kBlockOf<G>) void norm_forward_kernel(Norm<E, WT> g) {
  constexpr int W = kVec<E>, kRows = kBlockOf<G> / G;
  __shared__ float2 s_sum[G > 64 ? G / 64 : 1];
  const int lane = threadIdx.x % G;
  const float inv = 1.f / static_cast<float>(g.D);
  float w[NV][W], b[NV][W];
  load_weights<WT, NV, W, G>(g.weight, g.D, lane, 1.f, w);
  load_weights<WT, NV, W, G>(g.bias, g.D, lane, 0.f, b);
  for (long long r = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / G; r < g.rows;
       r += static_cast<long long>(gridDim.x) * kRows) {
    float v[NV][W], total = 0.f;
    {
      E raw[NV][W], res[NV][W];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * G + lane) * W;
        if (at < g.D) load_part(g.x + r * g.ld_x + at, g.D - at, raw[j]);
        if (at < g.D && g.residual != nullptr) load_part(g.residual + r * g.ld_res + at, g.D - at, res[j]);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * G + lane) * W;
        if (at < g.D && g.residual != nullptr) {
#pragma unroll
          for (int k = 0; k < W; ++k) raw[j][k] = from_f<E>(to_f(raw[j][k]) + to_f(res[j][k]));
          store_part(g.sum + r * g.D + at, g.D - at, raw[j]);
        }
#pragma unroll
        for (int k = 0; k < W; ++k) {
          v[j][k] = at < g.D ? to_f(raw[j][k]) : 0.f;
          total += v[j][k];
        }
      }
    }
    const float mean = row_sums<G>(total, 0.f, s_sum).x / static_cast<float>(g.D);
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
      E out[W];
#pragma unroll
      for (int k = 0; k < W; ++k) out[k] = from_f<E>(fmaf((v[j][k] - row.rest) * row.rstd, w[j][k], b[j][k]));
      if (at < g.D) store_part(g.y + r * g.D + at, g.D - at, out);
    }
  }
}

template <class E, class WT, int G, int NV>
__global__ __launch_bounds__(kBlockOf<G>) void norm_backward_kernel(Norm<E, WT> g) {
  constexpr int W = kVec<E>, kRows = kBlockOf<G> / G;
  __shared__ float2 s_sum[G > 64 ? G / 64 : 1];
  __shared__ float s_part[G <= 64 ? 2 : 1][G <= 64 ? G * NV * W : 1];
  const int lane = threadIdx.x % G;
  const float inv = 1.f / static_cast<float>(g.D);
  float w[NV][W], dw[NV][W], db[NV][W];
  load_weights<WT, NV, W, G>(g.weight, g.D, lane, 1.f, w);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < W; ++k) dw[j][k] = db[j][k] = 0.f;
  for (long long r = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / G; r < g.rows;
       r += static_cast<long long>(gridDim.x) * kRows) {
    E s[NV][W], gy[NV][W], gs[NV][W];
    const float mean = g.mean[r], rstd = g.rstd[r];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * G + lane) * W;
      if (at < g.D) {
        load_part(g.x + r * g.ld_x + at, g.D - at, s[j]);
        load_part(g.gy + r * g.ld_gy + at, g.D - at, gy[j]);
        if (g.gs != nullptr) load_part(g.gs + r * g.ld_gs + at, g.D - at, gs[j]);
      }
    }
    float m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if ((j * G + lane) * W + k >= g.D) continue;
        const float n = (to_f(s[j][k]) - mean) * rstd, o = to_f(gy[j][k]), q = o * w[j][k];
        dw[j][k] = fmaf(o, n, dw[j][k]);
        db[j][k] += o;
        m1 += q;
        m2 = fmaf(q, n, m2);
      }
    const float2 m = row_sums<G>(m1, m2, s_sum);
    m1 = m.x * inv;
    m2 = m.y * inv;
    if (g.gx != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * G + lane) * W;
        if (at >= g.D) continue;
        E out[W];
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const float n = (to_f(s[j][k]) - mean) * rstd;
          const float d = rstd * (fmaf(-n, m2, to_f(gy[j][k]) * w[j][k] - m1));
          out[k] = from_f<E>(g.gs != nullptr ? d + to_f(gs[j][k]) : d);
        }
        store_part(g.gx + r * g.D + at, g.D - at, out);
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
      store_part(part + at, g.D - at, dw[j]);
      store_part(part + g.D + at, g.D - at, db[j]);
    }
  }
}

// Rows longer than a workgroup's registers hold: the same sums in three passes over the row.
template <class E, class WT>
__global__ __launch_bounds__(kMaxThreads) void long_forward_kernel(Norm<E, WT> g) {
  __shared__ float2 s_sum[kMaxThreads / 64];
  const float inv = 1.f / static_cast<float>(g.D);
  for (long long r = blockIdx.x; r < g.rows; r += gridDim.x) {
    const E* in = g.x + r * g.ld_x;
    if (g.residual != nullptr) {
      for (int i = threadIdx.x; i < g.D; i += kMaxThreads)
        g.sum[r * g.D + i] = from_f<E>(to_f(in[i]) + to_f(g.residual[r * g.ld_res + i]));
      in = g.sum + r * g.D;  // a thread reads back its own elements
    }
    float total = 0.f;
    for (int i = threadIdx.x; i < g.D; i += kMaxThreads) total += to_f(in[i]);
    const float mean = row_sums<kMaxThreads>(total, 0.f, s_sum).x / static_cast<float>(g.D);
    float square = 0.f, rest = 0.f;
    for (int i = threadIdx.x; i < g.D; i += kMaxThreads) {
      const float c = to_f(in[i]) - mean;
      square = fmaf(c, c, square);
      rest += c;
    }
    const Row row = row_of(row_sums<kMaxThreads>(square, rest, s_sum), inv, g.eps);
    if (threadIdx.x == 0 && g.mean != nullptr) {
      g.mean[r] = mean + row.rest;
      g.rstd[r] = row.rstd;
    }
    for (int i = threadIdx.x; i < g.D; i += kMaxThreads)
      g.y[r * g.D + i] = from_f<E>(fmaf((to_f(in[i]) - mean - row.rest) * row.rstd, g.weight != nullptr ? to_f(g.weight[i]) : 1.f,
                                        g.bias != nullptr ? to_f(g.bias[i]) : 0.f));
  }
}

template <class E, class WT>
__global__ __launch_bounds__(kMaxThreads) void long_backward_kernel(Norm<E, WT> g) {
  __shared__ float2 s_sum[kMaxThreads / 64];
  const float inv = 1.f / static_cast<float>(g.D);
  for (long long r = blockIdx.x; r < g.rows; r += gridDim.x) {
    const E* s = g.x + r * g.ld_x;
    const E* gy = g.gy + r * g.ld_gy;
    const float mean = g.mean[r], rstd = g.rstd[r];
    float m1 = 0.f, m2 = 0.f;
    for (int i = threadIdx.x; i < g.D; i += kMaxThreads) {
      const float q = to_f(gy[i]) * (g.weight != nullptr ? to_f(g.weight[i]) : 1.f);
      m1 += q;
      m2 = fmaf(q, (to_f(s[i]) - mean) * rstd, m2);
    }
    const float2 m = row_sums<kMaxThreads>(m1, m2, s_sum);
    for (int i = threadIdx.x; i < g.D; i += kMaxThreads) {
      const float q = to_f(gy[i]) * (g.weight != nullptr ? to_f(g.weight[i]) : 1.f);
      const float d = rstd * fmaf(-(to_f(s[i]) - mean) * rstd, m.y * inv, q - m.x * inv);
      g.gx[r * g.D + i] = from_f<E>(g.gs != nullptr ? d + to_f(g.gs[r * g.ld_gs + i]) : d);
    }
  }
}

// dw and db of such rows: a workgroup's rows, 64 columns a wave.
template <class E, class WT>
__global__ __launch_bounds__(kThreads) void long_columns_kernel(Norm<E, WT> g, int n_parts) {
  const int n_cols = (g.D + kThreads - 1) / kThreads;
  const int part = static_cast<int>(blockIdx.x) / n_cols, i = static_cast<int>(blockIdx.x) % n_cols * kThreads + threadIdx.x;
  if (i >= g.D) return;
  float dw = 0.f, db = 0.f;
  for (long long r = part; r < g.rows; r += n_parts) {
    const float o = to_f(g.gy[r * g.ld_gy + i]);
    dw = fmaf(o, (to_f(g.x[r * g.ld_x + i]) - g.mean[r]) * g.rstd[r], dw);
    db += o;
  }
  float* out = g.partial + static_cast<size_t>(part) * 2 * g.D;
  out[i] = dw;
  out[g.D + i] = db;
}

// dw and db from n partial sums: a column takes 16 rows of lanes, each every sixteenth
// partial sum, in 64 bits.
template <class WT>
__global__ __launch_bounds__(kMaxThreads) void norm_sum_kernel(const float* partial, int n, int D, WT* dw, WT* db) {
  __shared__ double s_sum[kMaxThreads / 64][64];
  const long long cols = 2ll * D, i = static_cast<long long>(blockIdx.x) * 64 + threadIdx.x % 64;
  const int w = threadIdx.x / 64;
  double t = 0;
  if (i < cols)
    for (int r = w; r < n; r += kMaxThreads / 64) t += partial[r * cols + i];
  s_sum[w][threadIdx.x % 64] = t;
  __syncthreads();
  if (w != 0 || i >= cols) return;
  for (int v = 1; v < kMaxThreads / 64; ++v) t += s_sum[v][threadIdx.x];
  WT* out = i < D ? dw : db;
  if (out != nullptr) out[i < D ? i : i - D] = from_f<WT>(static_cast<float>(t));
}

// Calls f(G, NV) with the least group that holds D elements, or returns false.
template <class E, class F>
bool with_group(int64_t D, F f) {
  constexpr int W = kVec<E>;
  using std::integral_constant;
#define OSSM_GROUP(G, NV) \
  if (D <= int64_t(G) * (NV) * W) return f(integral_constant<int, G>{}, integral_constant<int, NV>{}), true
  OSSM_GROUP(8, 1);
  OSSM_GROUP(16, 1);
  OSSM_GROUP(32, 1);
  OSSM_GROUP(64, 1);
  OSSM_GROUP(64, 2);
  OSSM_GROUP(64, 4);
  OSSM_GROUP(256, 2);
  OSSM_GROUP(256, 4);
  OSSM_GROUP(1024, (sizeof(E) == 2 ? 2 : 4));
#undef OSSM_GROUP
  return false;
}

// Workgroups that walk the rows: as many as the card holds at once.
int64_t walkers(int64_t rows, int rows_each, int threads, int cus, int waves) {
  const int64_t most = int64_t(cus > 0 ? cus : 256) * (waves * 64 / threads > 0 ? waves * 64 / threads : 1);
  const int64_t need = (rows + rows_each - 1) / rows_each;
  return need < most ? need : most;
}

constexpr int kForwardWaves = 32, kBackwardWaves = 12;  // a CU

template <class E, class WT>
int forward(Norm<E, WT> g, int cus, hipStream_t st) {
  const bool held = with_group<E>(g.D, [&](auto G, auto NV) {
    constexpr int kG = decltype(G)::value, kNV = decltype(NV)::value, kB = kBlockOf<kG>;
    hipLaunchKernelGGL((norm_forward_kernel<E, WT, kG, kNV>),
                       dim3(static_cast<unsigned>(walkers(g.rows, kB / kG, kB, cus, kForwardWaves))), dim3(kB), 0, st, g);
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
  const bool held = with_group<E>(g.D, [&](auto G, auto) {
    constexpr int kG = decltype(G)::value, kB = kBlockOf<kG>;
    parts = walkers(g.rows, kB / kG, kB, cus, kBackwardWaves);
  });
  const int n_cols = (g.D + kThreads - 1) / kThreads;
  if (!held) parts = walkers(g.rows, 64, kThreads, cus, 16 / (n_cols < 16 ? n_cols : 16));
  const bool sums = dw != nullptr || db != nullptr;
  if (sums) {
    void* p = nullptr;
    if (int rc = acquire_workspace(call, static_cast<size_t>(parts) * 2 * g.D * sizeof(float), &p)) return rc;
    g.partial = static_cast<float*>(p);
  }
  with_group<E>(g.D, [&](auto G, auto NV) {
    constexpr int kG = decltype(G)::value, kNV = decltype(NV)::value, kB = kBlockOf<kG>;
    hipLaunchKernelGGL((norm_backward_kernel<E, WT, kG, kNV>), dim3(static_cast<unsigned>(parts)), dim3(kB), 0, st, g);
  });
  if (!held) {
    if (g.gx != nullptr)
      hipLaunchKernelGGL((long_backward_kernel<E, WT>),
                         dim3(static_cast<unsigned>(walkers(g.rows, 1, kMaxThreads, cus, kForwardWaves))), dim3(kMaxThreads),
                         0, st, g);
    if (sums) {
      if (int rc = check_grid("layer_norm_backward", parts * n_cols, kThreads)) return rc;
      hipLaunchKernelGGL((long_columns_kernel<E, WT>), dim3(static_cast<unsigned>(parts * n_cols)), dim3(kThreads), 0, st, g,
                         static_cast<int>(parts));
    }
  }
  if (int rc = launch_check("norm_backward_kernel")) return rc;
  if (!sums) return OSSM_OK;
  hipLaunchKernelGGL(norm_sum_kernel<WT>, dim3(static_cast<unsigned>((2ll * g.D + 63) / 64)), dim3(kMaxThreads), 0, st,
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
