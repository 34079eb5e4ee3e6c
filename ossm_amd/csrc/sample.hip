// The choice of the next token from a row of logits and a given random number
// (ossm_sample_logits): temperature, top-k, top-p and min-p.
//
//   w_v = exp((l_v - max) / T)
//   kept, in falling order of l (equal ones by index): the first k; of those each before
//   which less than p of their sum lies; of those each with w_v >= m; the first always
//   token = least v at which the sum of kept weights up to it passes u times all
//
// Weights are 64-bit whole numbers, w_v 2^S rounded, S from 46 down by the vocabulary's
// size so that no sum overflows: integer sums do not depend on their order, so the
// answer does not depend on how the row is cut, and a result next to a border
// is the exact one but for the weights' own rounding.  In float32 the sums' error of some 1e-7 times the
// 1e5 borders of a vocabulary would move one row in a hundred to a neighbouring token.  The
// exponential is 2^y = 2^(j/64) 2^e e^r, a table and five terms in 64 bits (error 2^-50):
// ten instructions, at the rate of float32's.
//
// A workgroup takes a row, in passes over it (from the caches after the first).  Logits are
// compared by their bits as an unsigned number in their order (a key).  The first pass finds
// the largest.  Where top-k or top-p is set, the next counts the row (or sums its weights) in
// 2048 bins of equal width below the largest, which gives the bin in which the last kept token lies;
// that bin's tokens are gathered in LDS, sorted, and give the last kept key and how many of
// the tokens that share it are kept, the first by index.  Where all that top-k keeps
// fits LDS the row is not looked at again.  Else a last pass sums the kept weights by stretches of
// 512 entries, and the one that passes the target is looked at entry by entry.  A bin that does not fit (a row
// of mostly equal logits) is cut by the keys' bits instead, in up to three further rounds (select).
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

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWavesOf = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 4096, kPer = kList / kThreads;  // gathered tokens, and a thread's
constexpr int kEach = 8;                              // consecutive entries of a lane
constexpr int kStretch = 64 * kEach;                  // entries of a wave at a time
constexpr int kMaxVocab = 1 << 20;
constexpr int kStretches = kMaxVocab / kStretch;

__constant__ double kPowers[64] = {  // 2^(j / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,};

struct Sample {
  const float* uniform;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  long long ld, rows;
  int V, scale;  // weights are multiples of 2^-scale
};

// The bits of a logit as an unsigned number in the logits' order; -0 is 0, and NaN is -inf.
constexpr uint32_t kLowest = 0x007fffffu;  // -inf
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l != l ? -__builtin_inff() : l + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A row's weights.  top: the largest logit's key.
struct Weights {
  const double* powers;  // in LDS
  double top, rate;      // rate = log2(e) / T
  int scale;
  bool infinite;         // the largest is +inf: it shares the answer with its like alone

  // w 2^scale
  __device__ __forceinline__ double scaled(uint32_t key) const {
    if (infinite) return key == 0xff800000u ? ldexp(1., scale) : 0.;
    const double y = (static_cast<double>(value_of(key)) - top) * rate;
    if (key == kLowest || !(y > -64.)) return 0.;  // below half a unit
    const double t = y + 0x1.8p46;                 // y to the nearest 64th, its 64ths in the low bits
    const int n = static_cast<int>(static_cast<uint32_t>(__double_as_longlong(t)));
    const double r = (y - (t - 0x1.8p46)) * 0.69314718055994530942;
    double s = 1. / 120.;
    s = fma(s, r, 1. / 24.);
    s = fma(s, r, 1. / 6.);
    s = fma(s, r, 0.5);
    s = fma(s, r, 1.);
    const double p = powers[n & 63];
    return ldexp(fma(p * r, s, p), (n >> 6) + scale);
  }
  static __device__ __forceinline__ u64 whole(double w) {  // to nearest
    return static_cast<u64>(__double_as_longlong(w + 0x1p52)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 of(uint32_t key) const { return whole(scaled(key)); }
};

// floor(f v) or, with up, the next whole number where it is none, for 0 <= f < 1.
__device__ __forceinline__ u64 part_of(float f, u64 v, bool up) {
  if (!(f > 0.f)) return 0;
  const uint32_t b = __float_as_uint(f);
  const int e = static_cast<int>(b >> 23);
  const u64 m = e == 0 ? b & 0x7fffffu : (b & 0x7fffffu) | 0x800000u;
  const int s = e == 0 ? 149 : 150 - e;  // f = m 2^-s, s >= 24
  const u64 lo = m * v, hi = __umul64hi(m, v);
  u64 q, rest;
  if (s < 64) {
    q = hi << (64 - s) | lo >> s;
    rest = lo << (64 - s);
  } else if (s < 128) {
    q = s == 64 ? hi : hi >> (s - 64);
    rest = lo | (s == 64 ? 0 : hi << (128 - s));
  } else {
    q = 0;
    rest = lo | hi;
  }
  return q + (up && rest != 0 ? 1 : 0);
}

// What is kept of a row: every key above `key`, and of those equal to it the first `ties`
// by index.
struct Kept {
  uint32_t key;
  uint32_t ties, same;  // of `same` tokens
  u64 weight;           // of all kept
};

struct Shared {
  double powers[64];
  u64 wave_weight[kWavesOf];
  uint32_t wave_count[kWavesOf];
  u64 weight_before;
  uint32_t bin, count_before, listed, above, same;
  int at;
  union {
    struct {
      u64 weight[kBins];
      uint32_t count[kBins];
    };
    struct {
      u64 item[kList], item_weight[kList];
    };
    struct {
      u64 stretch[kStretches];
      uint32_t ties[kStretches];
      uint32_t kept[kWavesOf][kStretch];
    };
  };
};

// f(index, key) of every entry of the row, in any order; four vectors a thread are asked for
// at once (one at a time a pass was bound by their latency).
template <class E, class F>
__device__ __forceinline__ void each_key(const E* row, int V, F f) {
  constexpr int kAhead = 4, kStep = kThreads * kEach;
  for (int at0 = static_cast<int>(threadIdx.x) * kEach; at0 < V; at0 += kAhead * kStep) {
    Vec<E, kEach> v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = at0 + u * kStep;
      v[u].zero();
      if (at < V) v[u].load(row + at, V - at);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = at0 + u * kStep;
      if (at >= V) break;
#pragma unroll
      for (int k = 0; k < kEach; ++k)
        if (at + k < V) f(at + k, key_of(v[u].get(k)));
    }
  }
}

// Inclusive sums over a workgroup's threads.
__device__ __forceinline__ void scan_threads(u64& w, uint32_t& n, Shared& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 a = __shfl_up(w, o);
    const uint32_t b = __shfl_up(n, o);
    if (lane >= o) w += a, n += b;
  }
  if (lane == 63) s.wave_weight[wave] = w, s.wave_count[wave] = n;
  __syncthreads();
  for (int v = 0; v < wave; ++v) w += s.wave_weight[v], n += s.wave_count[v];
  __syncthreads();
}

// The bin, from the first, at whose end `count` and `weight` before the first have grown to n or
// w (kBins: none); what lies before it in s, the weight of all bins in *all.
__device__ __forceinline__ uint32_t last_bin(uint32_t count, u64 weight, u64 n, u64 w, u64* all, Shared& s) {
  constexpr int kPerBin = kBins / kThreads;
  u64 sw = 0, mine_w[kPerBin];
  uint32_t sn = 0, mine_n[kPerBin];
#pragma unroll
  for (int k = 0; k < kPerBin; ++k) {
    mine_w[k] = s.weight[threadIdx.x * kPerBin + k];
    mine_n[k] = s.count[threadIdx.x * kPerBin + k];
    sw += mine_w[k];
    sn += mine_n[k];
  }
  if (threadIdx.x == 0) s.bin = kBins;
  scan_threads(sw, sn, s);
  u64 end_w = weight + sw;
  uint32_t end_n = count + sn;
#pragma unroll
  for (int k = kPerBin - 1; k >= 0; --k) {
    const u64 before_w = end_w - mine_w[k];
    const uint32_t before_n = end_n - mine_n[k];
    if ((end_n >= n || end_w >= w) && before_n < n && before_w < w) {  // one thread's
      s.bin = threadIdx.x * kPerBin + k;
      s.count_before = before_n;
      s.weight_before = before_w;
    }
    end_w = before_w;
    end_n = before_n;
  }
  __syncthreads();
  u64 t = 0;
  for (int v = 0; v < kWavesOf; ++v) t += s.wave_weight[v];
  *all = t;
  return s.bin;
}

// The shortest run of tokens in falling order that has `n` tokens or the weight `w`
// (at least one unit), or the whole row.
template <class E>
__device__ Kept select(const E* row, int V, const Weights& wt, uint32_t top, uint32_t lowest, u64 n, u64 w, Shared& s) {
  uint32_t hi = top, lo = lowest;  // the key is among these
  u64 weight = 0;                  // of the keys above hi
  uint32_t count = 0;
  for (;;) {
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.weight[b] = 0, s.count[b] = 0;
    __syncthreads();
    each_key(row, V, [&](int, uint32_t key) {
      if (key <= hi && key >= lo) {
        const uint32_t b = (hi - key) >> shift;
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.weight[b], wt.of(key));
      }
    });
    __syncthreads();
    u64 all_w;
    const uint32_t bin = last_bin(count, weight, n, w, &all_w, s);
    if (bin == kBins) {  // everything
      __syncthreads();
      return {lowest, UINT_MAX, UINT_MAX, weight + all_w};
    }
    count = s.count_before;
    weight = s.weight_before;
    const uint32_t in_bin = s.count[bin];
    __syncthreads();
    hi = hi - (bin << shift);
    if (shift == 0) {
      const u64 each = wt.of(hi);
      u64 ties = n - count < in_bin ? n - count : in_bin;
      if (each > 0 && w - weight <= each * ties) ties = (w - weight + each - 1) / each;
      return {hi, static_cast<uint32_t>(ties), in_bin, weight + each * ties};
    }
    const uint32_t span = (1u << shift) - 1;
    lo = hi - lo > span ? hi - span : lo;
  }
}

// The row's bins: of equal width in the logits from the largest down, to where weights are
// nothing or the row ends.
struct Bins {
  float top, scale;
  __device__ __forceinline__ uint32_t of(uint32_t key) const {  // kBins and more: weighs nothing
    const float b = (top - value_of(key)) * scale;
    return b < static_cast<float>(kBins) ? static_cast<uint32_t>(b) : kBins;
  }
};

// s.item[0 .. n - 1] in falling order, n up to kList.
__device__ void sort_items(uint32_t n, Shared& s) {
  uint32_t size = 64;
  while (size < n) size *= 2;
  for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) s.item[i] = 0;
  __syncthreads();
  const bool alone = size <= 128;  // one wave's pairs
  if (!alone || threadIdx.x < 64) {
    for (uint32_t k = 2; k <= size; k *= 2) {
      for (uint32_t j = k / 2; j > 0; j /= 2) {
        for (uint32_t i = threadIdx.x; i < size / 2; i += kThreads) {
          const uint32_t a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 x = s.item[a], y = s.item[b];
          if (((a & k) == 0) != (x > y)) {
            s.item[a] = y;
            s.item[b] = x;
          }
        }
        if (alone) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else __syncthreads();
      }
    }
  }
  __syncthreads();
}

// Gathers the entries that `take` takes (key, index below it in order) as items; how many there
// are, of which at most kList are there.
template <class E, class F>
__device__ uint32_t gather(const E* row, int V, F take, Shared& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  each_key(row, V, [&](int at, uint32_t key) {
    if (take(key)) {
      const uint32_t i = atomicAdd(&s.listed, 1u);
      if (i < kList) s.item[i] = static_cast<u64>(key) << 32 | ~static_cast<uint32_t>(at);
    }
  });
  __syncthreads();
  const uint32_t n = s.listed;
  __syncthreads();
  return n;
}

// The weights of the first n sorted items as running sums (this thread's kPer from tid kPer on) on
// top of `before`; and the whole.
__device__ __forceinline__ u64 run_items(const Weights& wt, uint32_t n, u64 before, u64 (&sum)[kPer], Shared& s) {
  u64 w = 0;
  uint32_t none = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const uint32_t i = threadIdx.x * kPer + k;
    sum[k] = i < n ? wt.of(static_cast<uint32_t>(s.item[i] >> 32)) : 0;
    w += sum[k];
  }
  const u64 mine = w;
  scan_threads(w, none, s);
  u64 at = before + w - mine, all = before;
  for (int v = 0; v < kWavesOf; ++v) all += s.wave_weight[v];
#pragma unroll
  for (int k = 0; k < kPer; ++k) sum[k] = at += sum[k];
  return all;
}

// The first of n running sums that reaches `target`, n where none does.
__device__ __forceinline__ uint32_t first_reaching(const u64 (&sum)[kPer], uint32_t n, u64 target, Shared& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.at = static_cast<int>(n);
  __syncthreads();
#pragma unroll
  for (int k = kPer - 1; k >= 0; --k) {
    const uint32_t i = threadIdx.x * kPer + k;
    if (i < n && sum[k] >= target) atomicMin(&s.at, static_cast<int>(i));
  }
  __syncthreads();
  return static_cast<uint32_t>(s.at);
}

// What is kept where sorted item `at` of n is the last: a key that others share is kept up to it.
__device__ __forceinline__ Kept kept_to(uint32_t at, uint32_t n, Shared& s) {
  const uint32_t key = static_cast<uint32_t>(s.item[at] >> 32);
  if (threadIdx.x == 0) s.above = s.same = 0;
  __syncthreads();
  uint32_t above = 0, same = 0;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t k = static_cast<uint32_t>(s.item[i] >> 32);
    above += k > key;
    same += k == key;
  }
  if (above != 0) atomicAdd(&s.above, above);
  if (same != 0) atomicAdd(&s.same, same);
  __syncthreads();
  return {key, at + 1 - s.above, s.same, 0};
}

// The least key whose weight is at least `floor` (of keys from `lowest` to `top`, whose is): 64
// are tried at once.
__device__ __forceinline__ uint32_t key_of_floor(const Weights& wt, uint32_t lowest, uint32_t top, double floor) {
  uint32_t lo = lowest, hi = top;  // hi's weight reaches it
  const uint32_t lane = threadIdx.x & 63;
  while (lo < hi) {
    const uint32_t step = (hi - lo + 63) / 64, k = hi - lo > lane * step ? lo + lane * step : hi;
    const u64 reach = __ballot(wt.scaled(k) >= floor);
    if (reach == 0) {
      lo = min(hi, lo + 63 * step + 1);
      continue;
    }
    const int first = __builtin_ctzll(reach);
    hi = min(hi, lo + first * step);
    if (first > 0) lo += (first - 1) * step + 1;
  }
  return hi;
}

template <class E>
__global__ __launch_bounds__(kThreads) void sample_kernel(const E* logits, Sample g) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid / 64;
  const long long r = blockIdx.x;
  const E* row = logits + r * g.ld;
  const float T = g.temperature != nullptr ? g.temperature[r] : g.temperature_all;
  const int k_given = g.top_k != nullptr ? g.top_k[r] : g.top_k_all;
  const float p = g.top_p != nullptr ? g.top_p[r] : g.top_p_all, m = g.min_p != nullptr ? g.min_p[r] : g.min_p_all;
  const float u = g.uniform[r];
  if (tid < 64) s.powers[tid] = kPowers[tid];  // read after the next barrier

  // the largest logit, the first that has it, and the least but -inf
  u64 best = 0;
  uint32_t low = 0xffffffffu;
  each_key(row, g.V, [&](int at, uint32_t key) {
    const u64 b = static_cast<u64>(key) << 32 | ~static_cast<uint32_t>(at);
    best = b > best ? b : best;
    low = key > kLowest ? min(low, key) : low;
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 b = __shfl_xor(best, o);
    best = b > best ? b : best;
    low = min(low, static_cast<uint32_t>(__shfl_xor(static_cast<int>(low), o)));
  }
  if (lane == 0) s.wave_weight[wave] = best, s.wave_count[wave] = low;
  __syncthreads();
  for (int v = 0; v < kWavesOf; ++v) {
    best = s.wave_weight[v] > best ? s.wave_weight[v] : best;
    low = min(low, s.wave_count[v]);
  }
  __syncthreads();
  const uint32_t top = static_cast<uint32_t>(best >> 32);
  if (top == kLowest || !(T > 0.f)) {
    if (tid == 0) g.tokens[r] = top == kLowest ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(best));
    return;
  }
  const float max = value_of(top);
  const Weights wt{s.powers, max, 1.4426950408889634074 / T, g.scale, max == __builtin_inff()};
  const double floor = m > 0.f ? ldexp(static_cast<double>(m < 1.f ? m : 1.f), g.scale) : 0.;

  // keys below the lowest weigh nothing; those next to it may weigh nothing too
  const double least = static_cast<double>(max) - 45. * T;
  const uint32_t lowest = wt.infinite || !(least > -3.4028234e38) ? kLowest + 1 : key_of(static_cast<float>(least)) - 1;
  Kept kept{lowest, UINT_MAX, UINT_MAX, 0};
  const bool by_k = k_given > 0 && k_given < g.V, by_p = p < 1.f;
  const uint32_t k = static_cast<uint32_t>(k_given);
  // weights are nothing from 47.5 ln 2 T on
  const float range = fminf(max - value_of(low), 33.f * T) * 1.00001f;
  const bool even = !wt.infinite && range < 1e37f;  // else the bins' width is no number
  const Bins bins{max, range > 1e-30f ? static_cast<float>(kBins) / range : 0.f};

  if (by_k) {
    bool done = false;
    if (even) {
      for (int b = tid; b < kBins; b += kThreads) s.weight[b] = 0, s.count[b] = 0;
      __syncthreads();
      each_key(row, g.V, [&](int, uint32_t key) {
        const uint32_t b = bins.of(key);
        if (b < kBins) atomicAdd(&s.count[b], 1u);
      });
      __syncthreads();
      u64 all;
      const uint32_t bin = last_bin(0, 0, k, ~0ull, &all, s);
      done = bin == kBins;  // what weighs anything is fewer than k
      if (!done) {
        const uint32_t before = s.count_before, in_bin = s.count[bin];
        if (before + in_bin <= kList) {  // everything that is kept fits: no further pass
          const uint32_t n0 = gather(row, g.V, [&](uint32_t key) { return bins.of(key) <= bin; }, s);
          sort_items(n0, s);
          uint32_t n = min(k, n0);
          u64 sum[kPer];
          u64 total = run_items(wt, n, 0, sum, s);
          if (by_p) {
            const u64 part = part_of(p, total, true);
            n = min(n, first_reaching(sum, n, part > 0 ? part : 1, s) + 1);
          }
          if (floor > 0.) {  // weights fall: the first that does not reach it
            if (tid == 0) s.at = static_cast<int>(n);
            __syncthreads();
#pragma unroll
            for (int q = kPer - 1; q >= 0; --q) {
              const uint32_t i = tid * kPer + q;
              if (i < n && wt.scaled(static_cast<uint32_t>(s.item[i] >> 32)) < floor) atomicMin(&s.at, static_cast<int>(i));
            }
            __syncthreads();
            n = static_cast<uint32_t>(s.at) > 0 ? s.at : 1;
          }
          // the kept ones by their index
          u64 mine[kPer];
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const uint32_t i = tid * kPer + q;
            mine[q] = i < n ? s.item[i] : 0;
          }
          __syncthreads();
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const uint32_t i = tid * kPer + q;
            if (i < n) s.item[i] = mine[q] << 32 | mine[q] >> 32;  // ~index above the key: falling order is rising index
          }
          sort_items(n, s);
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const uint32_t i = tid * kPer + q;
            mine[q] = i < n ? s.item[i] : 0;
          }
          __syncthreads();
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const uint32_t i = tid * kPer + q;
            if (i < n) s.item[i] = mine[q] << 32 | mine[q] >> 32;
          }
          __syncthreads();
          total = run_items(wt, n, 0, sum, s);
          const u64 target = u < 1.f ? part_of(u, total, false) : total - 1;
          const uint32_t at = first_reaching(sum, n, target + 1, s);
          if (tid == 0) g.tokens[r] = static_cast<int64_t>(~static_cast<uint32_t>(s.item[at]));
          return;
        }
        if (in_bin <= kList) {
          const uint32_t n0 = gather(row, g.V, [&](uint32_t key) { return bins.of(key) == bin; }, s);
          sort_items(n0, s);
          kept = kept_to(k - before - 1, n0, s);
          done = true;
        }
        __syncthreads();
      }
    }
    if (!done) kept = select(row, g.V, wt, top, lowest, k, ~0ull, s);
  }
  if (by_p) {
    bool done = false;
    u64 part = 0;
    const bool some = kept.ties < kept.same;  // the last key's weight counts `ties` times
    if (even) {
      for (int b = tid; b < kBins; b += kThreads) s.weight[b] = 0, s.count[b] = 0;
      __syncthreads();
      each_key(row, g.V, [&](int, uint32_t key) {
        if (key > kept.key || (key == kept.key && !some)) {
          const uint32_t b = bins.of(key);
          if (b < kBins) atomicAdd(&s.weight[b], wt.of(key));
        }
      });
      if (some && tid == 0) atomicAdd(&s.weight[min(bins.of(kept.key), kBins - 1u)], wt.of(kept.key) * kept.ties);
      __syncthreads();
      u64 all;
      last_bin(0, 0, ~0ull, ~0ull, &all, s);
      __syncthreads();
      part = part_of(p, all, true);
      part = part > 0 ? part : 1;
      const uint32_t bin = last_bin(0, 0, ~0ull, part, &all, s);
      const u64 before = s.weight_before;
      const uint32_t n0 = gather(row, g.V, [&](uint32_t key) { return bins.of(key) == bin; }, s);
      if (n0 <= kList) {
        sort_items(n0, s);
        u64 sum[kPer];
        run_items(wt, n0, before, sum, s);
        const uint32_t at = first_reaching(sum, n0, part, s);
        kept = kept_to(min(at, n0 - 1), n0, s);
        done = true;
      }
      __syncthreads();
    } else {
      if (!by_k) kept = select(row, g.V, wt, top, lowest, UINT_MAX, ~0ull, s);
      part = part_of(p, kept.weight, true);
      part = part > 0 ? part : 1;
    }
    if (!done) kept = select(row, g.V, wt, top, lowest, ~0ull, part, s);
  }
  if (floor > 0.) {
    const uint32_t key = key_of_floor(wt, lowest, top, floor);
    if (key > kept.key) kept = Kept{key, UINT_MAX, UINT_MAX, 0};
  }

  // the kept weights of each stretch, of equal last ones the first
  const int n_stretches = (g.V + kStretch - 1) / kStretch;
  const bool some = kept.ties < kept.same;
  if (some) {
    for (int st = wave; st < n_stretches; st += kWavesOf) {
      const int at = st * kStretch + lane * kEach;
      uint32_t n = 0;
      Vec<E, kEach> v;
      v.zero();
      if (at < g.V) v.load(row + at, g.V - at);
#pragma unroll
      for (int q = 0; q < kEach; ++q)
        if (at + q < g.V) n += key_of(v.get(q)) == kept.key;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
      if (lane == 0) s.ties[st] = n;
    }
    __syncthreads();
    if (wave == 0) {
      uint32_t base = 0;
      for (int s0 = 0; s0 < n_stretches; s0 += 64) {
        const uint32_t mine = s0 + lane < n_stretches ? s.ties[s0 + lane] : 0;
        uint32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t b = __shfl_up(sum, o);
          if (lane >= o) sum += b;
        }
        if (s0 + lane < n_stretches) s.ties[s0 + lane] = base + sum - mine;
        base += __shfl(sum, 63);
      }
    }
    __syncthreads();
  }
  // the keys of a stretch's entries of the lane, those that are not kept as the lowest
  const auto keys_of = [&](int st, const Vec<E, kEach>& v, uint32_t (&key)[kEach]) {
    const int at = st * kStretch + lane * kEach;
    uint32_t n = 0, before = 0;
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      key[q] = at + q < g.V ? key_of(v.get(q)) : kLowest;
      n += key[q] == kept.key;
    }
    if (some) {
      uint32_t sum = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t b = __shfl_up(sum, o);
        if (lane >= o) sum += b;
      }
      before = s.ties[st] + sum - n;
    }
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const bool last = key[q] == kept.key;
      if (key[q] < kept.key || (last && some && before >= kept.ties)) key[q] = kLowest;
      before += last;
    }
  };
  for (int st0 = wave; st0 < n_stretches; st0 += 4 * kWavesOf) {
    Vec<E, kEach> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (st0 + i * kWavesOf) * kStretch + lane * kEach;
      v[i].zero();
      if (at < g.V) v[i].load(row + at, g.V - at);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int st = st0 + i * kWavesOf;
      if (st >= n_stretches) break;
      uint32_t key[kEach], n = 0;
      keys_of(st, v[i], key);
      u64 sum = 0;
      // few kept ones are brought together first: a weight takes 25 operations, this six
#pragma unroll
      for (int q = 0; q < kEach; ++q) {
        const u64 take = __ballot(key[q] != kLowest);
        if (key[q] != kLowest) s.kept[wave][n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(take >> 32),
                                                __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(take), 0u))] = key[q];
        n += __popcll(take);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (uint32_t e = lane; e < n; e += 64) sum += wt.of(s.kept[wave][e]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      if (lane == 0) s.stretch[st] = sum;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  // one wave: the whole sum, the stretch that passes the target, the entry in it
  u64 total = 0;
  for (int st = lane; st < n_stretches; st += 64) total += s.stretch[st];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
  u64 target = u < 1.f ? part_of(u, total, false) : total - 1;
  int found = n_stretches - 1;
  for (int s0 = 0; s0 < n_stretches; s0 += 64) {
    const u64 mine = s0 + lane < n_stretches ? s.stretch[s0 + lane] : 0;
    u64 sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 a = __shfl_up(sum, o);
      if (lane >= o) sum += a;
    }
    const u64 past = __ballot(sum > target);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      target -= __shfl(sum - mine, at);
      found = s0 + at;
      break;
    }
    target -= __shfl(sum, 63);
  }
  Vec<E, kEach> v;
  v.zero();
  const int at = found * kStretch + lane * kEach;
  if (at < g.V) v.load(row + at, g.V - at);
  uint32_t key[kEach];
  keys_of(found, v, key);
  u64 w[kEach], sum = 0;
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    w[q] = key[q] != kLowest ? wt.of(key[q]) : 0;
    sum += w[q];
  }
  const u64 mine = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 a = __shfl_up(sum, o);
    if (lane >= o) sum += a;
  }
  const u64 past = __ballot(sum > target);
  if (past == 0 || lane != __builtin_ctzll(past)) return;
  target -= sum - mine;
  int q = 0;
  u64 acc = w[0];
#pragma unroll
  for (int t = 1; t < kEach; ++t)
    if (acc <= target) acc += w[t], q = t;
  g.tokens[r] = at + q;
}

}  // namespace
}  // namespace ossm

using namespace ossm;

extern "C" {

int ossm_sample_logits(int dtype, const void* logits, int64_t ld_logits, const float* uniform, const float* temperature,
                       float temperature_all, const int32_t* top_k, int64_t top_k_all, const float* top_p, float top_p_all,
                       const float* min_p, float min_p_all, int64_t* tokens, int64_t rows, int64_t vocab,
                       ossm_stream_t stream_v) {
  clear_error();
  if (dtype != OSSM_F32 && dtype != OSSM_BF16) return set_error(OSSM_ERR_INVALID_ARGUMENT, "sample_logits: unknown dtype");
  if (rows < 0 || vocab < 0) return set_error(OSSM_ERR_INVALID_ARGUMENT, "sample_logits: negative size");
  if (rows == 0) return OSSM_OK;
  if (vocab == 0) return set_error(OSSM_ERR_INVALID_ARGUMENT, "sample_logits: an empty vocabulary");
  if (vocab > kMaxVocab) return set_error(OSSM_ERR_UNSUPPORTED, "sample_logits: a vocabulary of more than 2^20");
  if (!logits || !uniform || !tokens) return set_error(OSSM_ERR_INVALID_ARGUMENT, "sample_logits: null pointer");
  if (int rc = check_grid("sample_logits", rows, kThreads)) return rc;
  int bits = 0;
  while ((int64_t(1) << bits) < vocab) ++bits;
  Sample g{uniform, temperature, top_k, top_p, min_p, tokens, temperature_all, top_p_all, min_p_all,
           static_cast<int>(top_k_all < 0 ? 0 : top_k_all > INT_MAX ? INT_MAX : top_k_all), ld_logits, rows,
           static_cast<int>(vocab), 63 - bits < 46 ? 63 - bits : 46};
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  if (dtype == OSSM_BF16)
    hipLaunchKernelGGL(sample_kernel<bf16_t>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, st,
                       static_cast<const bf16_t*>(logits), g);
  else
    hipLaunchKernelGGL(sample_kernel<float>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, st,
                       static_cast<const float*>(logits), g);
  return launch_check("sample_kernel");
}

}  // extern "C"
