// Penalties for repeated tokens, biases and a grammar's mask on a model's logits, in
// one pass over them (ossm_control_logits):
//
//   l = logits[v];  v seen in the history: l = l > 0 ? l / rep : l rep
//   l -= freq c + pres (c > 0)   c: v's count in the part after the prompt
//   l += bias of v;  l = -inf where the mask forbids v
//
// A workgroup takes a row's block of kBlock vocabulary entries.  It copies the block
// through the mask, without looking at a value; meanwhile it marks the row's biases
// and counts its history for that block in LDS, and then forms the marked entries'
// results, few against the vocabulary (doing all of it entry by entry took 45 instructions
// an entry, two thirds of the time at [256, 131072]).  Integer LDS atomics only (the highest
// bias index, a mark, counts): their order does not reach a result.  Every block of a row
// reads the row's history again, from L2: a few kB against the block's logits.
//
// Vectors of 16 bytes are aligned to the row's address, whatever its offset (a
// vocabulary of odd size puts every row at another one); the row's ends take single
// elements.

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <string>

#include "../../include/ossm_lm.h"
#include "lm_types.hpp"
#include "runtime.hpp"

namespace ossm {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 8192;  // vocabulary entries of a workgroup
constexpr int kAhead = 16;    // history loads in flight a thread
constexpr int kBiasInLds = 512;  // biases whose values are kept in LDS

// An entry's word in LDS.  Narrow: bias index + 1 in the upper half, set first (the
// largest wins), then the mark of one seen at all and the count; it serves
// histories below 2^15 tokens and up to 2^16 - 1 biases with one word an entry (32 KB:
// with the biases' values four workgroups a CU).  Wide: the mark and the count in a word,
// biases in a second.
template <bool WIDE>
struct Words {
  static constexpr uint32_t kSeen = WIDE ? 0x80000000u : 0x8000u;
  static constexpr uint32_t kCount = kSeen - 1;
  static constexpr int kWords = WIDE ? 2 * kBlock : kBlock;
};

template <class E>
__device__ __forceinline__ E minus_inf();
template <>
__device__ __forceinline__ float minus_inf<float>() { return -__builtin_inff(); }
template <>
__device__ __forceinline__ bf16_t minus_inf<bf16_t>() { return bf16_t{0xff80}; }

template <class E>
struct Logits {
  const E* in;
  E* out;
  const int32_t* history;
  const int32_t* lengths;
  const int32_t* prompts;
  const float* rep;
  const float* pres;
  const float* freq;
  const int32_t* bias_ids;
  const float* bias;
  const int32_t* allowed;
  long long ld_in, ld_out, ld_h, ld_b, ld_a;
  float rep_all, pres_all, freq_all;
  int V, H, n_bias, n_blocks;
};

template <class E, int W>
struct alignas(W * sizeof(E)) Pack {
  E v[W];
};

template <class E, bool WIDE>
__global__ __launch_bounds__(kThreads) void control_logits_kernel(Logits<E> g) {
  constexpr int W = 16 / static_cast<int>(sizeof(E));
  constexpr uint32_t kSeen = Words<WIDE>::kSeen, kCount = Words<WIDE>::kCount;
  extern __shared__ uint32_t s_word[];
  __shared__ float s_value[kBiasInLds];
  uint32_t* s_bias = WIDE ? s_word + kBlock : s_word;
  const int row = static_cast<int>(blockIdx.x / g.n_blocks);
  const int blk = static_cast<int>(blockIdx.x % g.n_blocks);
  const int tid = threadIdx.x;
  const E* in = g.in + row * g.ld_in;
  E* out = g.out + row * g.ld_out;
  // entry v of the row is entry v + shift of its 16-byte vectors
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(E) % W);
  const bool same = static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(E) % W) == shift;
  const int v0 = blk * kBlock - shift;  // the block's first entry, before the row's start in its first block
  const int n = min(kBlock, g.V - v0);
  if (n <= 0) return;  // the block that a shifted row may need
  const int lo = max(v0, 0), span = max(v0 + n - lo, 0);  // the entries that exist
  // everything from memory that the block needs is asked for before the first barrier: a
  // wait each for the history, the mask and the biases' values made three fourths of a
  // small call's time
  constexpr int kVecs = kBlock / (kThreads * W);
  Pack<E, W> p[kVecs];
  uint32_t mask[kVecs][2];
  const int32_t* allowed = g.allowed != nullptr ? g.allowed + row * g.ld_a : nullptr;
#pragma unroll
  for (int q = 0; q < kVecs; ++q) {
    const int i = (q * kThreads + tid) * W, v = v0 + i;
    if (v >= 0 && i + W <= n) p[q] = *reinterpret_cast<const Pack<E, W>*>(in + v);
    mask[q][0] = mask[q][1] = 0xffffffffu;
    if (allowed != nullptr && i < n) {
      mask[q][0] = static_cast<uint32_t>(allowed[max(v, 0) >> 5]);
      mask[q][1] = static_cast<uint32_t>(allowed[(min(v + W, g.V) - 1) >> 5]);
    }
  }
  const int len = g.lengths != nullptr ? min(max(g.lengths[row], 0), g.H) : g.H;
  const int first = g.prompts != nullptr ? min(max(g.prompts[row], 0), g.H) : 0;
  const int32_t* hist = g.history + row * g.ld_h;
  int id[kAhead];
  const auto history = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) id[k] = i0 + k * kThreads < len ? hist[i0 + k * kThreads] : -1;
  };
  history(tid);
  const float* bias = g.bias + row * g.ld_b;
  const int32_t* bias_ids = g.bias_ids + row * g.ld_b;
  int bias_id[kBiasInLds / kThreads];
#pragma unroll
  for (int k = 0; k < kBiasInLds / kThreads; ++k) {
    const int i = k * kThreads + tid;
    bias_id[k] = i < g.n_bias ? bias_ids[i] : -1;
    if (i < g.n_bias) s_value[i] = bias[i];
  }
  const float rep = g.rep != nullptr ? g.rep[row] : g.rep_all;
  const float pres = g.pres != nullptr ? g.pres[row] : g.pres_all;
  const float freq = g.freq != nullptr ? g.freq[row] : g.freq_all;

  for (int i = tid * 4; i < Words<WIDE>::kWords; i += kThreads * 4) *reinterpret_cast<uint4*>(s_word + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const auto mark_bias = [&](int i, int t) {
    if (t >= 0 && static_cast<unsigned>(t - lo) < static_cast<unsigned>(span))
      atomicMax(&s_bias[t - v0], static_cast<uint32_t>(i + 1) << (WIDE ? 0 : 16));
  };
#pragma unroll
  for (int k = 0; k < kBiasInLds / kThreads; ++k) mark_bias(k * kThreads + tid, bias_id[k]);
  for (int i = kBiasInLds + tid; i < g.n_bias; i += kThreads) mark_bias(i, bias_ids[i]);
  if (!WIDE && g.n_bias > 0) __syncthreads();
  for (int i0 = tid; i0 < len; i0 += kThreads * kAhead) {
    if (i0 != tid) history(i0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      // an id below zero is far outside as an unsigned number, and lo >= 0
      if (id[k] >= 0 && static_cast<unsigned>(id[k] - lo) < static_cast<unsigned>(span)) {
        if (i0 + k * kThreads >= first) atomicAdd(&s_word[id[k] - v0], 1u);
        else atomicOr(&s_word[id[k] - v0], kSeen);
      }
    }
  }

  __syncthreads();  // the marks are whole

  // the block through the mask: entry e's bit is bit e % 32 of the first word, or of the
  // second where it lies in another.  A thread's entries are the bits of a word, entry
  // (q kThreads + tid) W + k bit q W + k: it copies them and forms the marked ones itself,
  // and its second store to an entry follows its first without a wait.
  static_assert(kBlock == 32 * kThreads, "a thread's entries are the bits of a word");
  const E none = minus_inf<E>();
  uint32_t marked = 0;
#pragma unroll
  for (int q = 0; q < kVecs; ++q) {
    const int i = (q * kThreads + tid) * W, v = v0 + i;
    if (i >= n) break;
    const int first_word = max(v, 0) >> 5;
    uint32_t bits = 0, marks = 0;
#pragma unroll
    for (int k = 0; k < W; ++k)
      bits |= ((mask[q][((v + k) >> 5) != first_word ? 1 : 0] >> ((v + k) & 31)) & 1u) << k;
#pragma unroll
    for (int k = 0; k < W; k += 4) {
      uint4 w = *reinterpret_cast<const uint4*>(&s_word[i + k]);
      if constexpr (WIDE) {
        const uint4 b = *reinterpret_cast<const uint4*>(&s_bias[i + k]);
        w = make_uint4(w.x | b.x, w.y | b.y, w.z | b.z, w.w | b.w);
      }
      marks |= ((w.x != 0) | (w.y != 0) << 1 | (w.z != 0) << 2 | (w.w != 0) << 3) << k;
    }
    marked |= (marks & bits) << (q * W);
    if (v >= 0 && i + W <= n) {
#pragma unroll
      for (int k = 0; k < W; ++k) p[q].v[k] = (bits >> k) & 1 ? p[q].v[k] : none;
      if (same) {
        *reinterpret_cast<Pack<E, W>*>(out + v) = p[q];
      } else {
#pragma unroll
        for (int k = 0; k < W; ++k) out[v + k] = p[q].v[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (v + k >= 0 && i + k < n) out[v + k] = (bits >> k) & 1 ? in[v + k] : none;
    }
  }
  while (marked != 0) {
    constexpr int kBatch = 4;  // entries whose logits are asked for together
    int at[kBatch];
    float l[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int bit = marked != 0 ? __builtin_ctz(marked) : -1;
      marked &= marked - 1;
      at[k] = bit < 0 ? -1 : ((bit / W) * kThreads + tid) * W + bit % W;
      l[k] = at[k] >= 0 ? to_f(in[v0 + at[k]]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (at[k] < 0) continue;
      const uint32_t w = s_word[at[k]], b = WIDE ? s_bias[at[k]] : w >> 16;
      if (w & (kSeen | kCount)) {
        l[k] = l[k] > 0.f ? l[k] / rep : l[k] * rep;
        const uint32_t c = w & kCount;
        if (c != 0) l[k] -= freq * static_cast<float>(c) + pres;
      }
      if (b != 0) l[k] += b <= kBiasInLds ? s_value[b - 1] : bias[b - 1];
      out[v0 + at[k]] = from_f<E>(l[k]);
    }
  }
}

template <class E>
int run(Logits<E> g, int64_t rows, hipStream_t st) {
  constexpr int W = 16 / static_cast<int>(sizeof(E));
  g.n_blocks = (g.V + W - 1 + kBlock - 1) / kBlock;  // the shift may need one more
  if (rows > INT_MAX) return set_error(OSSM_ERR_UNSUPPORTED, "control_logits: size exceeds launch limits");
  if (int rc = check_grid("control_logits", rows * g.n_blocks, kThreads)) return rc;
  const bool wide = g.H >= (1 << 15) || g.n_bias >= (1 << 16);
  const size_t lds = (wide ? Words<true>::kWords : Words<false>::kWords) * sizeof(uint32_t);
  auto kern = wide ? control_logits_kernel<E, true> : control_logits_kernel<E, false>;
  if (wide)  // past 64 KB with the biases' values
    if (int rc = hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(lds)), "hipFuncSetAttribute"))
      return rc;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(rows * g.n_blocks)), dim3(kThreads), lds, st, g);
  return launch_check("control_logits_kernel");
}

}  // namespace
}  // namespace ossm

using namespace ossm;

extern "C" {

int ossm_control_logits(int dtype, const void* logits, int64_t ld_logits, void* out, int64_t ld_out,
                        const int32_t* history, int64_t ld_history, int64_t history_len,
                        const int32_t* lengths, const int32_t* prompt_lengths, const float* repetition,
                        float repetition_all, const float* presence, float presence_all,
                        const float* frequency, float frequency_all, const int32_t* bias_ids,
                        const float* bias_values, int64_t ld_bias, int64_t n_bias, const int32_t* allowed,
                        int64_t ld_allowed, int64_t rows, int64_t vocab, ossm_stream_t stream_v) {
  clear_error();
  if (dtype != OSSM_F32 && dtype != OSSM_BF16)
    return set_error(OSSM_ERR_INVALID_ARGUMENT, "control_logits: unknown dtype");
  if (rows < 0 || vocab < 0 || history_len < 0 || n_bias < 0)
    return set_error(OSSM_ERR_INVALID_ARGUMENT, "control_logits: negative size");
  if (vocab > INT_MAX / 2 || history_len > INT_MAX / 2 || n_bias > INT_MAX / 2)
    return set_error(OSSM_ERR_UNSUPPORTED, "control_logits: size exceeds launch limits");
  if (rows == 0 || vocab == 0) return OSSM_OK;
  if (!logits || !out || (history_len > 0 && !history) || (n_bias > 0 && (!bias_ids || !bias_values)))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, "control_logits: null pointer");
  if (rows > 1 && ld_out < vocab)
    return set_error(OSSM_ERR_INVALID_ARGUMENT, "control_logits: row stride of the output below the vocabulary");
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  const auto go = [&](auto e) {
    using E = decltype(e);
    return run(Logits<E>{static_cast<const E*>(logits), static_cast<E*>(out), history, lengths, prompt_lengths,
                         repetition, presence, frequency, bias_ids, bias_values, allowed, ld_logits, ld_out,
                         ld_history, ld_bias, ld_allowed, repetition_all, presence_all, frequency_all,
                         static_cast<int>(vocab), static_cast<int>(history_len), static_cast<int>(n_bias), 0},
               rows, st);
  };
  return dtype == OSSM_BF16 ? go(bf16_t{}) : go(0.f);
}

}  // extern "C"
