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
// exponential is 2^y = 2^(j/256) 2^e 2^f, a table and four terms in 64 bits (error 2^-52): some
// twenty operations, at the rate of float32's.
//
// A workgroup takes a row, in passes over it (from the caches after the first) that are bound by
// the operations an entry takes, not by memory: [256, 131072] in bf16 is 92 to 95 us, 14 at a copy's
// rate, and its slowest row's cycles are 20 thousand for the largest logit, 27 for the counts, 90 for
// the weights, 20 for the rest.  One row of 50001 takes 20 us.
//   top-k: of 1024 threads' own largest, the k-th is at least k logits' lower bound, and few more than
//     k reach it: those are gathered in LDS, sorted, and hold all that is kept; the row is not
//     looked at again.  For larger k (or where too many reach it) the row is counted in 8192 bins of equal
//     width below the largest first, which gives the bin of the k-th.
//   top-p: the counts by bins times the weights of the bins' middles tell about where the border is.
//     A pass then sums the weights, exactly, in all and by stretches of 512 entries above those
//     bins, and gathers the bins' tokens, which are sorted and give the last kept one.  The sums
//     tell whether it lies there at all.  Where min-p's border is above those bins, what min-p keeps is
//     summed instead, and is the answer if it is less than p's part.
//   Then the stretch that passes the target is looked at entry by entry; without top-p a pass
//     sums the stretches first.
// Where a bin's tokens do not fit (a row of mostly equal logits), or the border lies elsewhere (a p
// within 0.0006 of one: its bins are all of the row's tail, which on a large vocabulary no list holds), the
// last kept one is found by its bits, 11 at a time (select): such 256 rows of normal logits take 98 us at p
// 0.9, 127 at 0.9995, and of three different logits 900, whose atomics meet in a few digits.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <string>
#include <type_traits>

#include "../../include/ossm_lm.h"
#include "lm_types.hpp"
#include "lm_vector.hpp"
#include "runtime.hpp"

namespace ossm {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWavesOf = kThreads / 64;
constexpr int kBins = 8192, kPerBins = kBins / kThreads;
constexpr int kDigits = 2048;                         // of a round of select
constexpr int kList = 4096, kPer = kList / kThreads;  // gathered tokens, and a thread's
constexpr int kRanked = 256;                          // items sorted by their ranks alone
constexpr int kBuckets = kThreads, kCrowd = 512;      // where more are, and the most of one
constexpr int kEach = 8;                              // consecutive entries of a lane
constexpr int kStretch = 64 * kEach;                  // entries of a wave at a time
constexpr int kIndexBits = 20, kMaxVocab = 1 << kIndexBits;
constexpr int kStretches = kMaxVocab / kStretch;

__constant__ double kPowers[256] = {  // 2^(j / 256)
    1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175,
    1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738,
    1.0218971486541166, 1.0246677928971357, 1.0274459491187637, 1.030231637686041,
    1.0330248790212284, 1.0358256936019572, 1.0386341019613787, 1.041450124688316,
    1.0442737824274138, 1.0471050958792898, 1.0499440858006872, 1.0527907730046264,
    1.0556451783605572, 1.0585073227945128, 1.061377227289262, 1.0642549128844645,
    1.0671404006768237, 1.0700337118202419, 1.0729348675259756, 1.075843889062791,
    1.0787607977571199, 1.0816856149932152, 1.0846183622133092, 1.0875590609177697,
    1.0905077326652577, 1.0934643990728858, 1.0964290818163769, 1.099401802630222,
    1.102382583307841, 1.1053714457017412, 1.1083684117236787, 1.1113735033448175,
    1.1143867425958924, 1.1174081515673693, 1.1204377524096067, 1.12347556733302,
    1.1265216186082418, 1.129575928566288, 1.1326385195987192, 1.1357094141578055,
    1.1387886347566916, 1.1418762039695616, 1.1449721444318042, 1.148076478840179,
    1.1511892299529827, 1.154310420590216, 1.1574400736337511, 1.1605782120274988,
    1.1637248587775775, 1.1668800369524817, 1.1700437696832502, 1.1732160801636373,
    1.1763969916502812, 1.1795865274628758, 1.182784710984341, 1.1859915656609938,
    1.189207115002721, 1.1924313825831512, 1.1956643920398273, 1.1989061670743806,
    1.202156731452703, 1.2054161090051239, 1.2086843236265816, 1.2119613992768012,
    1.215247359980469, 1.2185422298274085, 1.2218460329727576, 1.2251587936371455,
    1.22848053610687, 1.2318112847340759, 1.2351510639369334, 1.2384998981998165,
    1.241857812073484, 1.245224830175258, 1.2486009771892048, 1.2519862778663162,
    1.255380757024691, 1.2587844395497165, 1.2621973503942507, 1.2656195145788063,
    1.2690509571917332, 1.2724917033894028, 1.275941778396392, 1.2794012075056693,
    1.2828700160787783, 1.2863482295460256, 1.2898358734066657, 1.2933329732290895,
    1.2968395546510096, 1.3003556433796506, 1.3038812651919358, 1.3074164459346773,
    1.3109612115247644, 1.3145155879493546, 1.318079601266064, 1.3216532776031575,
    1.3252366431597413, 1.3288297242059544, 1.3324325470831615, 1.3360451382041458,
    1.339667524053303, 1.3432997311868353, 1.3469417862329458, 1.3505937158920345,
    1.3542555469368927, 1.3579273062129011, 1.3616090206382248, 1.365300717204012,
    1.3690024229745905, 1.3727141650876684, 1.3764359707545302, 1.380167867260238,
    1.383909881963832, 1.387662042298529, 1.3914243757719262, 1.3951969099662003,
    1.3989796725383112, 1.4027726912202048, 1.4065759938190154, 1.4103896082172707,
    1.4142135623730951, 1.4180478843204152, 1.4218926021691656, 1.4257477441054942,
    1.42961333839197, 1.433489413367789, 1.4373759974489824, 1.4412731191286257,
    1.4451808069770467, 1.449099089642035, 1.4530279958490526, 1.4569675544014438,
    1.460917794180647, 1.4648787441464057, 1.4688504333369818, 1.4728328908693675,
    1.4768261459394993, 1.4808302278224719, 1.4848451658727524, 1.488870989524397,
    1.4929077282912648, 1.4969554117672355, 1.5010140696264256, 1.5050837316234065,
    1.5091644275934228, 1.5132561874526098, 1.5173590411982147, 1.5214730189088146,
    1.5255981507445384, 1.529734466947287, 1.533881997840956, 1.5380407738316568,
    1.5422108254079407, 1.5463921831410214, 1.550584877685, 1.5547889397770887,
    1.559004400237837, 1.5632312899713576, 1.567469639965553, 1.5717194812923414,
    1.5759808451078865, 1.5802537626528246, 1.5845382652524937, 1.588834384317164,
    1.593142151342267, 1.597461597908627, 1.6017927556826934, 1.606135656416771,
    1.6104903319492543, 1.6148568142048607, 1.6192351351948637, 1.6236253270173289,
    1.6280274218573478, 1.632441451987275, 1.6368674497669644, 1.6413054476440063,
    1.645755478153965, 1.6502175739206177, 1.6546917676561943, 1.6591780921616162,
    1.6636765803267364, 1.6681872651305825, 1.6727101796415966, 1.6772453570178785,
    1.681792830507429, 1.6863526334483934, 1.6909247992693053, 1.6955093614893326,
    1.7001063537185235, 1.7047158096580513, 1.709337763100463, 1.713972247929926,
    1.718619298122478, 1.723278947746274, 1.7279512309618377, 1.732636182022311,
    1.7373338352737062, 1.7420442251551564, 1.746767386199169, 1.7515033530318782,
    1.7562521603732995, 1.761013843037584, 1.7657884359332727, 1.7705759740635547,
    1.7753764925265212, 1.7801900265154245, 1.785016611318935, 1.789856282321401,
    1.7947090750031072, 1.7995750249405351, 1.804454167806624, 1.809346539371032,
    1.8142521755003989, 1.8191711121586085, 1.8241033854070534, 1.8290490314048973,
    1.8340080864093424, 1.8389805867758937, 1.843966568958626, 1.8489660695104508,
    1.8539791250833855, 1.8590057724288205, 1.864046048397789, 1.8690999899412386,
    1.8741676341103, 1.8792490180565602, 1.8843441790323345, 1.8894531543909392,
    1.8945759815869656, 1.8997126981765553, 1.9048633418176741, 1.9100279502703899,
    1.9152065613971474, 1.9203992131630474, 1.925605943636125, 1.930826790987627,
    1.9360617934922943, 1.9413109895286405, 1.9465744175792332, 1.9518521162309783,
    1.9571441241754002, 1.9624504802089273, 1.9677712232331759, 1.9731063922552343,
    1.978456026387951, 1.9838201648502194, 1.9891988469672663, 1.9945921121709402,
};

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

// A gathered token: its key, of which bfloat16's is 16 bits, over its index's complement, so that
// equal ones fall in rising order of index.
constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;
template <class E>
__device__ __forceinline__ u64 item_of(float l, uint32_t index) {
  return static_cast<u64>(sizeof(E) == 2 ? key_of(l) >> 16 : key_of(l)) << kIndexBits | (kIndexMask ^ index);
}
template <class E>
__device__ __forceinline__ uint32_t item_key(u64 item) {
  const uint32_t k = static_cast<uint32_t>(item >> kIndexBits);
  return sizeof(E) == 4 ? k : k << 16 | (k & 0x8000u ? 0u : 0xffffu);
}
__device__ __forceinline__ uint32_t item_index(u64 item) { return ~static_cast<uint32_t>(item) & kIndexMask; }

// A row's weights.
struct Weights {
  const __attribute__((address_space(3))) double* powers;  // a pointer to anywhere would make its loads slow
  double top, rate;      // the largest logit (finite), log2(e) / T
  int scale;

  // w 2^scale; NaN and -inf weigh nothing.  No branches: eight entries' chains of dependent
  // operations have to overlap (one at a time a pass took ten times as long).
  __device__ __forceinline__ double scaled(float v) const {
    const double y = fmax((static_cast<double>(v) - top) * rate, -64.);  // 2^-64: below half a unit
    const double t = y + 0x1.8p44;                 // y to the nearest 256th, its 256ths in the low bits
    const int n = static_cast<int>(static_cast<uint32_t>(__double_as_longlong(t)));
    const double f = y - (t - 0x1.8p44);           // (ln 2)^n / n!, f <= 2^-9: left out 2^-59
    double s = 9.6181291076284771619e-3;
    s = fma(s, f, 5.5504108664821579953e-2);
    s = fma(s, f, 2.4022650695910071233e-1);
    s = fma(s, f, 6.9314718055994530942e-1);
    const double p = powers[n & 255];
    return ldexp(fma(p * f, s, p), (n >> 8) + scale);
  }
  static __device__ __forceinline__ u64 whole(double w) {  // to nearest
    return static_cast<u64>(__double_as_longlong(w + 0x1p52)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 of(float v) const { return whole(scaled(v)); }
  __device__ __forceinline__ u64 of(uint32_t key) const { return of(value_of(key)); }
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
  double powers[256];
  u64 wave_weight[kWavesOf], wave_more[kWavesOf];
  uint32_t wave_count[kWavesOf];
  u64 weight_before;
  uint32_t bin, count_before, listed, above, same;
  int at;
  uint32_t bucket[kBuckets];
  u64 stretch[kStretches];
  union {
    uint32_t bins[kBins];
    struct {
      u64 weight[kDigits];
      uint32_t count[kDigits];
    };
    u64 item[kList];
    struct {
      uint32_t ties[kStretches];
      float kept[kWavesOf][kStretch];
    };
  };
};

// f(first index, values) of every vector of the row, by whole waves (a stretch each), -inf behind
// its end; four vectors a thread are asked for at once (one at a time a pass was bound by their
// latency).
template <class E, class F>
__device__ __forceinline__ void each_vector(const E* row, int V, F f) {
  constexpr int kAhead = 4, kStep = kThreads * kEach;
  const int lane_at = static_cast<int>(threadIdx.x & 63) * kEach;
  for (int st0 = static_cast<int>(threadIdx.x / 64) * kStretch; st0 < V; st0 += kAhead * kStep) {
    Vec<E, kEach> v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = st0 + u * kStep + lane_at;
      v[u].zero();
      if (at < V) v[u].load(row + at, V - at);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = st0 + u * kStep + lane_at;
      if (st0 + u * kStep >= V) break;
      float x[kEach];
#pragma unroll
      for (int k = 0; k < kEach; ++k) x[k] = v[u].get(k);
      if (at + kEach > V) {
#pragma unroll
        for (int k = 0; k < kEach; ++k)
          if (at + k >= V) x[k] = -__builtin_inff();
      }
      f(at, x);
    }
  }
}

// The sum over a wave, in its last lane, without a way through LDS.
__device__ __forceinline__ u64 sum_to_last(u64 v) {
#define OSSM_ADD(CTRL, ROWS)                                                                              \
  {                                                                                                       \
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);       \
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false); \
    v += static_cast<u64>(hi) << 32 | lo;                                                                 \
  }
  OSSM_ADD(0x111, 0xf)  // a row's lanes on by 1, 2, 4, 8
  OSSM_ADD(0x112, 0xf)
  OSSM_ADD(0x114, 0xf)
  OSSM_ADD(0x118, 0xf)
  OSSM_ADD(0x142, 0xa)  // the last of rows 0 and 2 to the next row
  OSSM_ADD(0x143, 0xc)  // the last of row 1 to rows 2 and 3
#undef OSSM_ADD
  return v;
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
#pragma unroll
  for (int v = 0; v < kWavesOf; ++v) {  // all are read, so that one does not wait for another
    const u64 a = s.wave_weight[v];
    const uint32_t b = s.wave_count[v];
    if (v < wave) w += a, n += b;
  }
  __syncthreads();
}

// The digit, from the first, at whose end `count` and `weight` before the first have grown to n or
// w (kDigits: none); what lies before it in s, the weight of all digits in *all.
__device__ __forceinline__ uint32_t last_digit(uint32_t count, u64 weight, u64 n, u64 w, u64* all, Shared& s) {
  constexpr int kPerDigit = kDigits / kThreads;
  u64 sw = 0, mine_w[kPerDigit];
  uint32_t sn = 0, mine_n[kPerDigit];
#pragma unroll
  for (int k = 0; k < kPerDigit; ++k) {
    mine_w[k] = s.weight[threadIdx.x * kPerDigit + k];
    mine_n[k] = s.count[threadIdx.x * kPerDigit + k];
    sw += mine_w[k];
    sn += mine_n[k];
  }
  if (threadIdx.x == 0) s.bin = kDigits;
  scan_threads(sw, sn, s);
  u64 end_w = weight + sw;
  uint32_t end_n = count + sn;
#pragma unroll
  for (int k = kPerDigit - 1; k >= 0; --k) {
    const u64 before_w = end_w - mine_w[k];
    const uint32_t before_n = end_n - mine_n[k];
    if ((end_n >= n || end_w >= w) && before_n < n && before_w < w) {  // one thread's
      s.bin = threadIdx.x * kPerDigit + k;
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
__device__ __forceinline__ Kept select(const E* row, int V, const Weights& wt, uint32_t top, uint32_t lowest, u64 n, u64 w, Shared& s) {
  uint32_t hi = top, lo = lowest;  // the key is among these
  u64 weight = 0;                  // of the keys above hi
  uint32_t count = 0;
  for (;;) {
    int shift = 0;
    while (((hi - lo) >> shift) >= kDigits) ++shift;
    __syncthreads();
    for (int b = threadIdx.x; b < kDigits; b += kThreads) s.weight[b] = 0, s.count[b] = 0;
    __syncthreads();
    each_vector(row, V, [&](int, const float (&x)[kEach]) {
#pragma unroll
      for (int q = 0; q < kEach; ++q) {
        const uint32_t key = key_of(x[q]);
        if (key > hi || key < lo) continue;
        const uint32_t b = (hi - key) >> shift;
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.weight[b], wt.of(x[q]));
      }
    });
    __syncthreads();
    u64 all_w;
    const uint32_t bin = last_digit(count, weight, n, w, &all_w, s);
    if (bin == kDigits) {  // everything
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

// The row's bins: of equal width in the logits from the largest down, to about where weights are
// nothing or the row ends; the last takes all below it down to `lowest`.  What lies lower weighs
// nothing and is in none, so that a bin's count is the number of entries from its start on.
struct Bins {
  float top, scale, lowest;
  __device__ __forceinline__ uint32_t of(float v) const {  // kBins: below `lowest`, -inf and NaN
    // the least of two is the number where the other is NaN: an infinite difference at scale 0
    return v >= lowest ? static_cast<uint32_t>(fminf((top - v) * scale, kBins - 1.f)) : kBins;
  }
};

__device__ __forceinline__ void clear_bins(Shared& s) {
  __syncthreads();
  for (int b = threadIdx.x * 4; b < kBins; b += kThreads * 4) *reinterpret_cast<uint4*>(s.bins + b) = make_uint4(0, 0, 0, 0);
  __syncthreads();
}

// The bin, of PER a thread, in which the n-th entry lies (kBins: there are fewer), s.count_before
// what lies before it.
template <int PER>
__device__ __forceinline__ uint32_t bin_of_count(uint32_t n, Shared& s) {
  uint32_t mine[PER], sum = 0;
  u64 none = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    mine[k] = s.bins[threadIdx.x * PER + k];
    sum += mine[k];
  }
  if (threadIdx.x == 0) s.bin = kBins;
  scan_threads(none, sum, s);
#pragma unroll
  for (int k = PER - 1; k >= 0; --k) {
    const uint32_t before = sum - mine[k];
    if (sum >= n && before < n) {
      s.bin = threadIdx.x * PER + k;
      s.count_before = before;
    }
    sum = before;
  }
  __syncthreads();
  return s.bin;
}

// The bins between which the p-th part of the weight is reached, as far as the bins' counts and
// the weights of their middles tell.
__device__ __forceinline__ void bins_of_part(const Weights& wt, const Bins& bins, float p, uint32_t& first, uint32_t& last, Shared& s) {
  constexpr float kUnit = 16777216.f;  // 2^24
  // a middle's weight may be off by half a bin, 0.2 percent, but most bins' errors cancel; where
  // they do not, the border is found by bits.  Four times this gathered 4200 tokens at p = 0.98 of
  // 131072 normal logits, more than a list holds
  constexpr float kMargin = 0.0006f;
  u64 mine[kPerBins], sum = 0;
  uint32_t none = 0;
  const float step = bins.scale > 0.f ? static_cast<float>(wt.rate) / bins.scale : 0.f;
#pragma unroll
  for (int k = 0; k < kPerBins; ++k) {
    const uint32_t b = threadIdx.x * kPerBins + k;
    mine[k] = static_cast<u64>(static_cast<float>(s.bins[b]) * kUnit * __builtin_amdgcn_exp2f(-(static_cast<float>(b) + 0.5f) * step));
    sum += mine[k];
  }
  if (threadIdx.x == 0) s.count_before = kBins - 1, s.bin = kBins - 1;
  scan_threads(sum, none, s);
  u64 all = 0;
  for (int v = 0; v < kWavesOf; ++v) all += s.wave_weight[v];
  const float part = p * static_cast<float>(all);
  const u64 least = static_cast<u64>(fmaxf(part - kMargin * static_cast<float>(all), 0.f)) + 1;
  const u64 most = static_cast<u64>(part + kMargin * static_cast<float>(all)) + 1;
#pragma unroll
  for (int k = kPerBins - 1; k >= 0; --k) {
    const u64 before = sum - mine[k];
    if (sum >= least && before < least) s.count_before = threadIdx.x * kPerBins + k;
    if (sum >= most && before < most) s.bin = threadIdx.x * kPerBins + k;
    sum = before;
  }
  __syncthreads();
  first = s.count_before;
  last = s.bin;
}

// The least key, of those from `lo` to `hi`, that is `in` with all above it (hi is): 64 are
// tried at once, by every wave alike.
template <class F>
__device__ __forceinline__ uint32_t least_key(uint32_t lo, uint32_t hi, F in) {
  const uint32_t lane = threadIdx.x & 63;
  while (lo < hi) {
    const uint32_t step = (hi - lo + 63) / 64, k = hi - lo > lane * step ? lo + lane * step : hi;
    const u64 reach = __ballot(in(value_of(k)));
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

// s.item[0 .. n - 1] in falling order, n up to PER a thread, no two alike.  Up to kRanked of them by
// counting the larger ones of each (64 items a wave, the others shared among the waves): few barriers,
// 2000 cycles at 5 items, 10000 at 226.  More of them first go to 1024 buckets of equal width between
// the largest and the least (12000 at 5, 13000 at 226), and are ranked in their own.  Where many share
// one, they take a sorting network (17000 at 224, 43000 at 1123); a wave's pairs lie in 128
// neighbouring items while they are up to 64 apart, and need no other wave.
template <int PER>
__device__ __forceinline__ void sort_items(uint32_t n, Shared& s) {
  const uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid & 63;
  if (n <= 1) return;
  if (n <= kRanked) {
    const uint32_t blocks = (n + 63) / 64, slices = kWavesOf / blocks;
    const uint32_t i = wave % blocks * 64 + lane, slice = wave / blocks;
    const u64 own = i < n ? s.item[i] : 0;
    if (tid < kRanked) s.bucket[tid] = 0;
    __syncthreads();
    if (slice < slices) {
      uint32_t larger = 0;
      for (uint32_t j = slice; j < n; j += 4 * slices) {
        u64 other[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) other[q] = j + q * slices < n ? s.item[j + q * slices] : 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) larger += other[q] > own;
      }
      if (i < n) atomicAdd(&s.bucket[i], larger);
    }
    __syncthreads();
    const u64 mine = tid < n ? s.item[tid] : 0;
    __syncthreads();
    if (tid < n) s.item[s.bucket[tid]] = mine;
    __syncthreads();
    return;
  }
  u64 mine[PER], hi = 0, lo = ~0ull;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const uint32_t i = tid + q * kThreads;
    mine[q] = i < n ? s.item[i] : 0;
    if (i >= n) continue;
    hi = hi > mine[q] ? hi : mine[q];
    lo = lo < mine[q] ? lo : mine[q];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 a = __shfl_xor(hi, o), b = __shfl_xor(lo, o);
    hi = hi > a ? hi : a;
    lo = lo < b ? lo : b;
  }
  if (lane == 0) s.wave_weight[wave] = hi, s.wave_more[wave] = lo;
  s.bucket[tid] = 0;
  __syncthreads();
  for (int v = 0; v < kWavesOf; ++v) {
    hi = hi > s.wave_weight[v] ? hi : s.wave_weight[v];
    lo = lo < s.wave_more[v] ? lo : s.wave_more[v];
  }
  const int shift = max(54 - __clzll(static_cast<long long>(hi - lo)), 0);  // hi > lo: ten bits stay
  uint32_t place[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (tid + q * kThreads < n) place[q] = atomicAdd(&s.bucket[(hi - mine[q]) >> shift], 1u);
  __syncthreads();
  uint32_t own = s.bucket[tid], end = own;
  if (!__syncthreads_or(own > kCrowd)) {
    u64 none = 0;
    scan_threads(none, end, s);
    s.bucket[tid] = end - own;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q)
      if (tid + q * kThreads < n) s.item[s.bucket[(hi - mine[q]) >> shift] + place[q]] = mine[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (tid + q * kThreads >= n) continue;
      const uint32_t b = static_cast<uint32_t>((hi - mine[q]) >> shift);
      const uint32_t from = s.bucket[b], to = b + 1 < kBuckets ? s.bucket[b + 1] : n;
      place[q] = from;
      for (uint32_t j = from; j < to; j += 4) {
        u64 other[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) other[t] = j + t < to ? s.item[j + t] : 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) place[q] += other[t] > mine[q];
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q)
      if (tid + q * kThreads < n) s.item[place[q]] = mine[q];
    __syncthreads();
    return;
  }
  uint32_t size = 64;
  while (size < n) size *= 2;
  for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) s.item[i] = 0;
  __syncthreads();
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
      if (j > 64 || (j == 1 && k > 64)) __syncthreads();
      else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  __syncthreads();
}

// Gathers the entries from lo to below `end` (or all above where there is no end) as items; how
// many there are, of which at most kList are there.  f sees every vector, by whole waves.
template <class E, class F>
__device__ __forceinline__ uint32_t gather(const E* row, int V, float lo, float end, bool no_end, Shared& s, F f) {
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  each_vector(row, V, [&](int at, const float (&x)[kEach]) {
    f(at, x);
    uint32_t bits = 0;
#pragma unroll
    for (int q = 0; q < kEach; ++q) bits |= (x[q] >= lo && (no_end || x[q] < end) ? 1u : 0u) << q;
    if (bits == 0) return;
    uint32_t i = atomicAdd(&s.listed, static_cast<uint32_t>(__popc(bits)));
    while (bits != 0) {  // seldom more than one a lane
      const int t = __builtin_ctz(bits);
      float v = x[0];
#pragma unroll
      for (int q = 1; q < kEach; ++q) v = t == q ? x[q] : v;
      if (i < kList) s.item[i] = item_of<E>(v, static_cast<uint32_t>(at + t));
      ++i;
      bits &= bits - 1;
    }
  });
  __syncthreads();
  const uint32_t n = s.listed;
  __syncthreads();
  return n;
}

// The weights of the first n sorted items as running sums (this thread's PER from tid PER on, `first`
// the one before them) on top of `before`; and the whole.
template <class E, int PER>
__device__ __forceinline__ u64 run_items(const Weights& wt, uint32_t n, u64 before, u64 (&sum)[PER], u64& first, Shared& s) {
  u64 w = 0;
  uint32_t none = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const uint32_t i = threadIdx.x * PER + k;
    sum[k] = i < n ? wt.of(item_key<E>(s.item[i])) : 0;
    w += sum[k];
  }
  const u64 mine = w;
  scan_threads(w, none, s);
  u64 at = first = before + w - mine, all = before;
  for (int v = 0; v < kWavesOf; ++v) all += s.wave_weight[v];
#pragma unroll
  for (int k = 0; k < PER; ++k) sum[k] = at += sum[k];
  return all;
}

// The first of n running sums that reaches `target`, which lies above what the first starts from;
// n where none does.
template <int PER>
__device__ __forceinline__ uint32_t first_reaching(const u64 (&sum)[PER], u64 first, uint32_t n, u64 target, Shared& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.at = static_cast<int>(n);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const uint32_t i = threadIdx.x * PER + k;
    if (i < n && sum[k] >= target && first < target) s.at = static_cast<int>(i);  // one thread's
    first = sum[k];
  }
  __syncthreads();
  return static_cast<uint32_t>(s.at);
}

// What is kept where sorted item `at` of n is the last: a key that others share is kept up to it.
template <class E>
__device__ __forceinline__ Kept kept_to(uint32_t at, uint32_t n, Shared& s) {
  const uint32_t key = item_key<E>(s.item[at]);
  if (threadIdx.x == 0) s.above = s.same = 0;
  __syncthreads();
  uint32_t above = 0, same = 0;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t k = item_key<E>(s.item[i]);
    above += k > key;
    same += k == key;
  }
  if (above != 0) atomicAdd(&s.above, above);
  if (same != 0) atomicAdd(&s.same, same);
  __syncthreads();
  return {key, at + 1 - s.above, s.same, 0};
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
  if (tid < 256) s.powers[tid] = kPowers[tid];  // read after the next barrier
  const bool by_k = k_given > 0 && k_given < g.V, by_p = p < 1.f;

  // the largest logit (of the thread's own in mine) and about the least but -inf, of every
  // eighth.  The median of x, y and +inf is the larger, or y where x is NaN.
  float mine = -__builtin_inff(), low = __builtin_inff();
  const bool by_threads = by_k && k_given <= kThreads && k_given <= (g.V + kEach - 1) / kEach;
  each_vector(row, g.V, [&](int, const float (&x)[kEach]) {
#pragma unroll
    for (int q = 0; q < kEach; ++q) mine = __builtin_amdgcn_fmed3f(x[q], mine, __builtin_inff());
    low = __builtin_amdgcn_fmed3f(x[0] > -__builtin_inff() ? x[0] : __builtin_inff(), low, -__builtin_inff());
  });
  float max = mine;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    max = fmaxf(max, __shfl_xor(max, o));
    low = fminf(low, __shfl_xor(low, o));
  }
  if (lane == 0) s.kept[wave][0] = max, s.kept[wave][1] = low;
  __syncthreads();
  for (int v = 0; v < kWavesOf; ++v) {
    max = fmaxf(max, s.kept[v][0]);
    low = fminf(low, s.kept[v][1]);
  }
  __syncthreads();
  max += 0.f;  // -0 is 0
  if (max == -__builtin_inff()) {
    if (tid == 0) g.tokens[r] = -1;
    return;
  }
  if (!(T > 0.f)) {  // the first that is the largest
    if (tid == 0) s.at = INT_MAX;
    __syncthreads();
    int first = INT_MAX;
    each_vector(row, g.V, [&](int at, const float (&x)[kEach]) {
#pragma unroll
      for (int q = 0; q < kEach; ++q)
        if (x[q] == max) first = min(first, at + q);
    });
    if (first < INT_MAX) atomicMin(&s.at, first);
    __syncthreads();
    if (tid == 0) g.tokens[r] = s.at;
    return;
  }
  asm volatile("" ::"v"(u));  // here already: where it is used it would be waited for
  const uint32_t top = key_of(max);
  const bool infinite = max == __builtin_inff();  // it shares the answer with its like alone
  const Weights wt{(const __attribute__((address_space(3))) double*)s.powers, max, 1.4426950408889634074 / T, g.scale};
  const double floor = m > 0.f ? ldexp(static_cast<double>(m < 1.f ? m : 1.f), g.scale) : 0.;

  // keys below the lowest weigh nothing; those next to it may weigh nothing too
  const double least = static_cast<double>(max) - 45. * T;
  const uint32_t lowest = infinite || !(least > -3.4028234e38) ? kLowest + 1 : key_of(static_cast<float>(least)) - 1;
  Kept kept{lowest, UINT_MAX, UINT_MAX, 0};
  const uint32_t k = by_k ? static_cast<uint32_t>(k_given) : UINT_MAX;
  // weights are nothing from 47.5 ln 2 T on
  const float range = fminf(low < max ? max - low : __builtin_inff(), 33.f * T) * 1.00001f;
  const bool even = range < 1e37f;  // else the bins' width is no number
  const Bins bins{max, range > 1e-30f ? static_cast<float>(kBins) / range : 0.f, value_of(lowest)};
  const auto bin_start = [&](uint32_t b) {  // the least value of bin b and those before
    return value_of(least_key(lowest, top, [&](float v) { return bins.of(v) <= b; }));
  };

  // all that can be kept as items: the k largest and what few lie near the last, or a short row
  uint32_t listed = UINT_MAX;
  bool all_kept = false;  // what weighs anything is fewer than k
  if (infinite) {  // equal weights: the first of them, as many as k and p leave
    if (tid == 0) s.same = 0;
    __syncthreads();
    uint32_t n = 0;
    each_vector(row, g.V, [&](int, const float (&x)[kEach]) {
#pragma unroll
      for (int q = 0; q < kEach; ++q) n += x[q] == max;
    });
    atomicAdd(&s.same, n);
    __syncthreads();
    kept = Kept{top, min(k, s.same), s.same, 0};
    if (by_p) kept.ties = static_cast<uint32_t>(part_of(p, kept.ties, true)) | (p > 0.f ? 0u : 1u);
  } else if ((by_k || by_p) && g.V <= kThreads) {
    listed = gather(row, g.V, -3.402823466e38f, 0.f, true, s, [](int, const float (&)[kEach]) {});
  } else if (by_k && even) {
    if (by_threads) {
      // eight bins in one: a bin a thread
      __syncthreads();
      s.bins[tid] = 0;
      __syncthreads();
      const uint32_t b = bins.of(mine);
      if (b < kBins) atomicAdd(&s.bins[b / kPerBins], 1u);
      __syncthreads();
      const uint32_t bin = bin_of_count<1>(k, s);
      if (bin < kBins)
        listed = gather(row, g.V, bin_start(bin * kPerBins + kPerBins - 1), 0.f, true, s, [](int, const float (&)[kEach]) {});
    }
    if (listed > kList) {
      clear_bins(s);
      each_vector(row, g.V, [&](int, const float (&x)[kEach]) {
#pragma unroll
        for (int q = 0; q < kEach; ++q) {
          const uint32_t b = bins.of(x[q]);
          if (b < kBins) atomicAdd(&s.bins[b], 1u);
        }
      });
      __syncthreads();
      const uint32_t bin = bin_of_count<kPerBins>(k, s);
      all_kept = bin == kBins;
      if (!all_kept) {
        const uint32_t before = s.count_before, in_bin = s.bins[bin];
        if (before + in_bin <= kList) {
          listed = gather(row, g.V, bin_start(bin), 0.f, true, s, [](int, const float (&)[kEach]) {});
        } else if (in_bin <= kList) {
          const uint32_t n0 = gather(row, g.V, bin_start(bin), bin > 0 ? bin_start(bin - 1) : 0.f, bin == 0, s,
                                     [](int, const float (&)[kEach]) {});
          sort_items<kPer>(n0, s);
          kept = kept_to<E>(k - before - 1, n0, s);
          all_kept = true;
        }
      }
    }
  }
  // the answer from the list, PER items a thread
  const auto from_list = [&](auto per) {
    constexpr int PER = decltype(per)::value;
    sort_items<PER>(listed, s);
    uint32_t n = min(k, listed);
    u64 sum[PER], first;
    u64 total = run_items<E, PER>(wt, n, 0, sum, first, s);
    if (by_p) {
      const u64 part = part_of(p, total, true);
      n = min(n, first_reaching<PER>(sum, first, n, part > 0 ? part : 1, s) + 1);
    }
    if (floor > 0.) {  // weights fall: the first that does not reach it
      __syncthreads();
      if (tid == 0) s.at = static_cast<int>(n);
      __syncthreads();
#pragma unroll
      for (int q = PER - 1; q >= 0; --q) {
        const uint32_t i = tid * PER + q;
        if (i < n && wt.scaled(value_of(item_key<E>(s.item[i]))) < floor) atomicMin(&s.at, static_cast<int>(i));
      }
      __syncthreads();
      n = s.at > 0 ? static_cast<uint32_t>(s.at) : 1u;
    }
    // the kept ones by their index: its complement above the key, so that falling order is rising index
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kThreads) s.item[i] = (s.item[i] & kIndexMask) << 32 | s.item[i] >> kIndexBits;
    __syncthreads();
    sort_items<PER>(n, s);
    for (uint32_t i = tid; i < n; i += kThreads) s.item[i] = s.item[i] << 32 >> (32 - kIndexBits) | s.item[i] >> 32;
    __syncthreads();
    total = run_items<E, PER>(wt, n, 0, sum, first, s);
    const u64 target = u < 1.f ? part_of(u, total, false) : total - 1;
    const uint32_t at = first_reaching<PER>(sum, first, n, target + 1, s);
    if (tid == 0) g.tokens[r] = item_index(s.item[at]);
  };
  if (listed <= kThreads) {
    from_list(std::integral_constant<int, 1>{});
    return;
  }
  if (listed <= kList) {
    from_list(std::integral_constant<int, kPer>{});
    return;
  }
  if (by_k && !all_kept && !infinite) kept = select(row, g.V, wt, top, lowest, k, ~0ull, s);

  const uint32_t floor_key =
      floor > 0. && !infinite ? least_key(lowest, top, [&](float v) { return wt.scaled(v) >= floor; }) : 0;
  uint32_t summed = 0;  // so many tokens are gathered, and the stretches' kept weights known
  if (by_p && !infinite) {
    const bool some = kept.ties < kept.same;  // the last key's weight counts `ties` times
    const float last = value_of(kept.key);
    u64 part = 0;
    bool done = false;
    if (even) {
      clear_bins(s);
      const float from = some ? value_of(kept.key + 1) : last;  // the least whose like are all kept
      each_vector(row, g.V, [&](int, const float (&x)[kEach]) {
#pragma unroll
        for (int q = 0; q < kEach; ++q) {
          const uint32_t b = bins.of(x[q]);
          if (b < kBins && x[q] >= from) atomicAdd(&s.bins[b], 1u);
        }
      });
      if (some && tid == 0) atomicAdd(&s.bins[min(bins.of(last), kBins - 1u)], kept.ties);
      __syncthreads();
      uint32_t b0, b1;
      bins_of_part(wt, bins, p, b0, b1, s);
      const float end = b0 > 0 ? bin_start(b0 - 1) : 0.f;
      // Sure to be kept: past the gathered ones.  Where min-p keeps fewer, what it keeps, and p's
      // border is not looked for if that is below p's part.
      const bool fewer = b0 > 0 && floor_key > 0 && value_of(floor_key) >= fmaxf(end, from);
      const float over = fewer ? value_of(floor_key) : b0 > 0 ? fmaxf(end, from) : __builtin_inff();
      u64 above = 0, total = 0;
      const uint32_t n0 = gather(row, g.V, fewer ? __builtin_inff() : bin_start(b1), end, b0 == 0, s, [&](int at, const float (&x)[kEach]) {
        u64 high = 0;
#pragma unroll
        for (int q = 0; q < kEach; ++q) {
          u64 w = wt.of(x[q]);
          asm volatile("" : "+v"(w));  // formed for every entry, not behind a branch for each
          total += x[q] >= from ? w : 0;
          high += x[q] >= over ? w : 0;
        }
        above += high;
        if (__ballot(high != 0) != 0) high = sum_to_last(high);
        if (lane == 63) s.stretch[at / kStretch] = high;
      });
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        total += __shfl_xor(total, o);
        above += __shfl_xor(above, o);
      }
      if (lane == 0) s.wave_weight[wave] = total, s.wave_more[wave] = above;
      __syncthreads();
      total = above = 0;
      for (int v = 0; v < kWavesOf; ++v) total += s.wave_weight[v], above += s.wave_more[v];
      __syncthreads();
      if (some) {  // its own bin or one behind: never above the gathered ones but where all are
        const u64 w = wt.of(last) * kept.ties;
        total += w;
        above += b0 > 0 && !fewer && last >= end ? w : 0;
      }
      part = part_of(p, total, true);
      part = part > 0 ? part : 1;
      if (fewer) {
        done = above < part;
        if (done) {
          kept = Kept{floor_key, UINT_MAX, UINT_MAX, 0};
          summed = 1;  // no last one is left out
        }
      } else if (n0 <= kList && above < part) {
        if (n0 <= kThreads) sort_items<1>(n0, s);
        else sort_items<kPer>(n0, s);
        u64 sum[kPer], first;
        run_items<E, kPer>(wt, n0, above, sum, first, s);
        const uint32_t at = first_reaching<kPer>(sum, first, n0, part, s);
        if (at < n0) {
          if (!some) {  // the gathered tokens' weights join those above them
            for (uint32_t i = tid; i <= at; i += kThreads) {
              const uint32_t key = item_key<E>(s.item[i]);
              if (key >= floor_key) atomicAdd(&s.stretch[item_index(s.item[i]) / kStretch], wt.of(key));
            }
            summed = n0;
          }
          kept = kept_to<E>(at, n0, s);
          done = true;
        }
        __syncthreads();
      }
    } else {
      if (!by_k) kept = select(row, g.V, wt, top, lowest, UINT_MAX, ~0ull, s);
      part = part_of(p, kept.weight, true);
      part = part > 0 ? part : 1;
    }
    if (!done) kept = select(row, g.V, wt, top, lowest, ~0ull, part, s);
  }
  if (floor_key > kept.key) kept = Kept{floor_key, UINT_MAX, UINT_MAX, 0};

  // the kept weights of each stretch, of equal last ones the first; the latter's numbers before each
  const int n_stretches = (g.V + kStretch - 1) / kStretch;
  const bool some = kept.ties < kept.same;
  const float last = value_of(kept.key);
  const auto load = [&](int st, Vec<E, kEach>& v) {
    const int at = st * kStretch + lane * kEach;
    v.zero();
    if (at < g.V) v.load(row + at, g.V - at);
  };
  __syncthreads();
  if (some && summed == 0) {
    for (int st = wave; st < n_stretches; st += kWavesOf) {
      Vec<E, kEach> v;
      load(st, v);
      uint32_t n = 0;
#pragma unroll
      for (int q = 0; q < kEach; ++q) n += st * kStretch + lane * kEach + q < g.V && v.get(q) == last;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
      if (lane == 0) s.ties[st] = n;
    }
    __syncthreads();
    if (wave == 0) {
      uint32_t base = 0;
      for (int s0 = 0; s0 < n_stretches; s0 += 64) {
        const uint32_t mine_n = s0 + lane < n_stretches ? s.ties[s0 + lane] : 0;
        uint32_t sum = mine_n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t b = __shfl_up(sum, o);
          if (lane >= o) sum += b;
        }
        if (s0 + lane < n_stretches) s.ties[s0 + lane] = base + sum - mine_n;
        base += __shfl(sum, 63);
      }
    }
    __syncthreads();
  }
  // which of the lane's entries of a stretch are kept, as bits, with so many of the last before it
  const auto kept_of = [&](int st, const Vec<E, kEach>& v, uint32_t ties) {
    const int left = g.V - (st * kStretch + lane * kEach);
    uint32_t bits = 0, same = 0;
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      bits |= (v.get(q) > last ? 1u : 0u) << q;
      same |= (v.get(q) == last ? 1u : 0u) << q;
    }
    const uint32_t in = left >= kEach ? 0xffu : left > 0 ? (1u << left) - 1 : 0u;
    bits &= in;
    same &= in;
    if (some) {
      const uint32_t n = __popc(same);
      uint32_t sum = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t b = __shfl_up(sum, o);
        if (lane >= o) sum += b;
      }
      const uint32_t before = ties + sum - n, room = before < kept.ties ? kept.ties - before : 0;
      while (static_cast<uint32_t>(__popc(same)) > room) same &= ~(0x80000000u >> __clz(same));  // the first ones stay
    }
    return bits | same;
  };
  for (int st0 = summed > 0 ? n_stretches : wave; st0 < n_stretches; st0 += 4 * kWavesOf) {
    Vec<E, kEach> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) load(min(st0 + i * kWavesOf, n_stretches - 1), v[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int st = st0 + i * kWavesOf;
      if (st >= n_stretches) break;
      const bool whole = !some && (st + 1) * kStretch <= g.V;  // no entry but by its value
      if (whole) {
        float most = -__builtin_inff();
#pragma unroll
        for (int q = 0; q < kEach; ++q) most = __builtin_amdgcn_fmed3f(v[i].get(q), most, __builtin_inff());
        if (__ballot(most >= last) == 0) {  // most stretches, where few tokens are kept
          if (lane == 0) s.stretch[st] = 0;
          continue;
        }
      }
      const uint32_t bits = whole ? 0 : kept_of(st, v[i], some ? s.ties[st] : 0);
      u64 sum = 0;
      uint32_t n = 0;
      // few kept ones are brought together first: a weight takes 25 operations, this six
#pragma unroll
      for (int q = 0; q < kEach; ++q) {
        const bool take = whole ? v[i].get(q) >= last : bits >> q & 1;
        const u64 takes = __ballot(take);
        if (take) s.kept[wave][n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(takes >> 32),
                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(takes), 0u))] = v[i].get(q);
        n += __popcll(takes);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (infinite) {
        sum = lane == 0 ? static_cast<u64>(n) << g.scale : 0;
      } else {
        for (uint32_t e = lane; e < n; e += 64) sum += wt.of(s.kept[wave][e]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      sum = sum_to_last(sum);
      if (lane == 63) s.stretch[st] = sum;
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
    const u64 own = s0 + lane < n_stretches ? s.stretch[s0 + lane] : 0;
    u64 sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 a = __shfl_up(sum, o);
      if (lane >= o) sum += a;
    }
    const u64 past = __ballot(sum > target);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      target -= __shfl(sum - own, at);
      found = s0 + at;
      break;
    }
    target -= __shfl(sum, 63);
  }
  Vec<E, kEach> v;
  load(found, v);
  uint32_t ties = 0;
  if (some && summed > 0) {
    for (uint32_t i = lane; i < summed; i += 64)
      ties += item_key<E>(s.item[i]) == kept.key && item_index(s.item[i]) < static_cast<uint32_t>(found) * kStretch;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ties += __shfl_xor(ties, o);
  } else if (some) {
    ties = s.ties[found];
  }
  const uint32_t bits = kept_of(found, v, ties);
  u64 w[kEach], sum = 0;
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    w[q] = (bits >> q & 1) == 0 ? 0 : infinite ? 1ull << g.scale : wt.of(v.get(q));
    sum += w[q];
  }
  const u64 own = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 a = __shfl_up(sum, o);
    if (lane >= o) sum += a;
  }
  const u64 past = __ballot(sum > target);
  if (past == 0) {  // nothing is kept: never, but a token is written on every path
    if (lane == 0) g.tokens[r] = -1;
    return;
  }
  if (lane != __builtin_ctzll(past)) return;
  target -= sum - own;
  int q = 0;
  u64 acc = w[0];
#pragma unroll
  for (int t = 1; t < kEach; ++t)
    if (acc <= target) acc += w[t], q = t;
  g.tokens[r] = found * kStretch + lane * kEach + q;
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
