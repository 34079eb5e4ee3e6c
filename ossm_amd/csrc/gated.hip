// The gated projection of a feed-forward block, forward and backward:
//
//   a = x Wg^T + bg,  b = x Wu^T + bu,  y = act(a) b
//   da = dy b act'(a),  db = dy act(a)
//   dx = da Wg + db Wu,  dWg = da^T x,  dWu = db^T x,  dbg = sum da,  dbu = sum db
//
// for row-major x [T, D], Wg, Wu [F, D], y [T, F].  One product kernel serves all of
// it: C(m, n) = sum_k A(m, k) B(n, k) of bf16 operands that lie either along k ("row":
// x and the weights in the forward, da and db in dx) or across it ("col": the weights in
// dx, both operands of dW).  Tiles go from memory straight into LDS, two buffers deep;
// operands across k are transposed by the LDS's transposing reads on their way to
// the matrix cores.  In the forward a tile's columns are half gate, half up rows of the
// same outputs, so that each wave holds a and b of an output in the same registers and
// the activation and product are its epilogue; training stores a and b (in float32) beside y,
// which the backward's elementwise kernel turns into da and db.
//
// float32: operands are split into three bf16 planes, x = x0 + x1 + x2, and the
// six products of order up to 2 are further stretches of k (split_mfma.hpp has the
// error).  A value that is not finite is held as (x, 0, 0), which makes NaN of sums
// where inf is due, so sums that are not finite are formed again on the fp32 matrix
// instruction from the planes' sums.
//
// bfloat16: da and db are rounded to bf16 between the elementwise kernel and the products
// (relative 2^-9, random; gradients then are 0.0024 off, where an exact sum rounded to
// bf16 is 0.0017 off and torch's bf16 steps, which round a, b, da and db, 0.0034 to
// 0.0039 at [8192, 2048] -> 8192), or, up to kTwoPlanes of them, held as two terms; sums
// are float32 throughout, and so are the stored a and b: in bf16 they left 0.0031.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <initializer_list>
#include <string>
#include <type_traits>
#include <utility>

#include "../../include/ossm_lm.h"
#include "lm_types.hpp"
#include "runtime.hpp"
#include "scan_device.hpp"
#include "split_mfma.hpp"

namespace ossm {
namespace {

constexpr int kOutside = 0x7ffffff0;  // a buffer offset past every range: the load gives zeros
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// ---- activations -------------------------------------------------------------
struct ActGrad {
  float f, d;  // act(a), act'(a)
};

template <int ACT>
__device__ __forceinline__ ActGrad activate(float a) {
  switch (ACT) {
    case OSSM_ACT_SILU: {
      const float s = sigmoid_f(a);
      return {a * s, s * (1.f + a * (1.f - s))};
    }
    case OSSM_ACT_SIGMOID: {
      const float s = sigmoid_f(a);
      return {s, s * (1.f - s)};
    }
    case OSSM_ACT_RELU: return {a > 0.f ? a : (a != a ? a : 0.f), a <= 0.f ? 0.f : 1.f};
    case OSSM_ACT_GELU: {
      const float cdf = 0.5f * (1.f + erff(a * 0.70710678118654752f));
      return {a * cdf, cdf + a * __expf(-0.5f * a * a) * 0.39894228040143268f};
    }
    default: {  // gelu, tanh form
      const float c = 0.79788456080286536f, k = 0.044715f;
      const float e = __expf(2.f * c * (a + k * a * a * a));
      const float t = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
      return {0.5f * a * (1.f + t), 0.5f * (1.f + t) + 0.5f * a * (1.f - t * t) * c * (1.f + 3.f * k * a * a)};
    }
  }
}

__device__ __forceinline__ float activation_of(int act, float a) {
  switch (act) {
    case OSSM_ACT_SILU: return activate<OSSM_ACT_SILU>(a).f;
    case OSSM_ACT_SIGMOID: return activate<OSSM_ACT_SIGMOID>(a).f;
    case OSSM_ACT_RELU: return activate<OSSM_ACT_RELU>(a).f;
    case OSSM_ACT_GELU: return activate<OSSM_ACT_GELU>(a).f;
    default: return activate<OSSM_ACT_GELU_TANH>(a).f;
  }
}

// ---- the product -------------------------------------------------------------
// Plane s of part p starts at p[part] + s * plane.  Row: element (i, k) at i ld + k; col:
// at k ld + i.  ld and every start are multiples of 8 elements (16 bytes).
struct Operand {
  const uint16_t* p[2];
  long long plane, ld;
};

template <class E>
struct Product {
  Operand a, b;
  int M, N, K;       // K: of one part
  int parts, combos; // stretches of k: parts x (1, or 2 or 6 products of planes)
  int tiles_m, tiles_n, splits, per_split;  // per_split: k tiles of one split
  // outputs
  E* c[2];           // plain: rows below `half` to c[0], from it on to c[1] (less half); gated: y in c[0]
  long long ldc;
  int half, half_rows;  // rows of each half that exist
  float* part;       // splits > 1: [splits][M][N]; gated: [splits][2][M][N]
  const E* bias[2];  // gated
  float* save[2];    // gated: a, b or null
  int act;
};

// products of planes, smallest first: (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
__device__ __forceinline__ int plane_a(int combo) { return (0x001012 >> (4 * combo)) & 3; }
__device__ __forceinline__ int plane_b(int combo) { return (0x010210 >> (4 * combo)) & 3; }

typedef __attribute__((address_space(3))) void lds_void;

// What the chunks of LDS row r of a row operand are turned by: eight neighbouring rows then
// put a k in eight places.
template <int TK>
__device__ __forceinline__ int row_turn(int r) { return TK == 64 ? r & 7 : (r >> 1) & 3; }

// The same for LDS row k of a col operand of R columns: the four k of a transposing read then
// lie in four stretches of 64 bytes.
template <int R>
__device__ __forceinline__ int col_turn(int k) { return R == 64 ? 4 * ((k >> 1) & 1) : 4 * (k & 3); }

// One operand's tiles of R rows (of m or n) and TK k into LDS.  An LDS row is TK k (row) or R
// columns (col) of 16-byte chunks; chunk c sits at c ^ row_turn (row) or c ^ col_turn
// (col), which spreads the fragments' reads over the banks.  A thread's chunks are the same
// in every tile, so their offsets are kept; chunks of rows past the matrix have one
// that the buffer's range turns into zeros, and the last tile of k masks its own.
template <bool COL, int R, int TK, int THREADS>
struct TileLoad {
  static constexpr int kRounds = R * (TK / 8) / THREADS, kChunks = R / 8;
  static_assert(!COL || R >= 64, "col_turn stays in a row");
  static constexpr int kRange = 0x40000000;  // every offset in a matrix is below it: 256 rows of 2^21 bytes
  int off[kRounds];

  // the chunk of its row that a thread's place in LDS holds (THREADS / 4 rows on: the same)
  static __device__ __forceinline__ int row_chunk() {
    const int tid = static_cast<int>(threadIdx.x);
    return (tid % (TK / 8)) ^ row_turn<TK>(tid / (TK / 8));
  }

  __device__ __forceinline__ void init(long long ld, int i0, int rows) {
    const int tid = static_cast<int>(threadIdx.x);
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int q = i * THREADS + tid;
      if constexpr (!COL) {
        const int r = q / (TK / 8), c = row_chunk();
        off[i] = i0 + r < rows ? static_cast<int>(r * ld * 2) + c * 16 : kOutside;
      } else {
        const int k = q / kChunks, c = (q % kChunks) ^ col_turn<R>(k);
        off[i] = i0 + c * 8 < rows ? static_cast<int>(k * ld * 2) + c * 16 : kOutside;
      }
    }
  }

  // round i of the tile at p, `left` k of it
  __device__ __forceinline__ void load(int i, uint16_t* lds, const uint16_t* p, int left) const {
    const int tid = static_cast<int>(threadIdx.x);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), 0, kRange, 0x00027000);
    const int k = COL ? (i * THREADS + tid) / kChunks : row_chunk() * 8;
    const int o = k < left ? off[i] : kOutside;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(lds + (i * THREADS + wave_id() * kWave) * 8), 16, o, 0, 0, 0);
  }
};

// The wave's fragment of 32 rows from i0 at k step kk (16 k) of a tile in LDS: lane l
// holds row l % 32 at k = 8 (l / 32) .. + 7.
template <bool COL, int R, int TK>
__device__ __forceinline__ bf16x8 load_frag(const uint16_t* lds, int i0, int kk) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  if constexpr (!COL) {
    const int r = i0 + (lane & 31), c = kk * 2 + (lane >> 5);
    return *reinterpret_cast<const bf16x8*>(lds + r * TK + ((c ^ row_turn<TK>(r)) * 8));
  } else {
    // a group of 16 lanes reads 4 k of 16 columns, transposed: lane i gets column i
    const int g = lane >> 4, i16 = lane & 15, kr = i16 >> 2;
    const int k = kk * 16 + (g >> 1) * 8 + kr, col = i0 + (g & 1) * 16 + (i16 & 3) * 4;
    const uint16_t* q = lds + k * R + (((col >> 3) ^ col_turn<R>(k)) * 8) + (col & 7);  // (of k + 4 too)
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)q);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(q + 4 * R));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// Element (i, k) of an operand as the sum of its planes, smallest first (0 outside).
template <bool COL>
__device__ __forceinline__ float element(const Operand& o, int planes, int part, int i, int rows, int k, int K) {
  if (i >= rows || k >= K) return 0.f;
  const uint16_t* p = o.p[part] + (COL ? static_cast<long long>(k) * o.ld + i : static_cast<long long>(i) * o.ld + k);
  float s = to_f(bf16_t{p[(planes - 1) * o.plane]});
  for (int j = planes - 2; j >= 0; --j) s += to_f(bf16_t{p[j * o.plane]});
  return s;
}

// Lays out a stretch of instructions: COUNT of a kind (0x100 LDS reads, 0x20 loads) spread
// over MFMA matrix instructions.
template <int KIND, int COUNT, int MFMA, int I = 0>
__device__ __forceinline__ void interleave() {
  constexpr int kGroups = COUNT < MFMA ? COUNT : MFMA;
  if constexpr (I < kGroups) {
    constexpr int kOfKind = (I + 1) * COUNT / kGroups - I * COUNT / kGroups;
    constexpr int kOfMfma = (I + 1) * MFMA / kGroups - I * MFMA / kGroups;
    __builtin_amdgcn_sched_group_barrier(KIND, kOfKind, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, kOfMfma, 0);
    interleave<KIND, COUNT, MFMA, I + 1>();
  }
}

// A tile's k and how many tiles LDS holds (one is read, the others are on their way): 64 and
// two where both operands are rows (whole 128-byte lines of each), 32 and three where one
// is not.  Both ways at [8192, 2048] -> 8192 in bf16, us: forward 480 and 520, dx 580 and
// 488, dW 584 and 553.
constexpr int tile_k(bool gated) { return gated ? 64 : 32; }
constexpr int tile_stages(bool gated) { return gated ? 2 : 3; }

// Workgroup tile: WM x WN waves of FM x FN fragments of 32 x 32.  GATED: the tile's
// columns are 32-column pairs, gate and up rows of the same outputs (N counts outputs).
//
// Bound by the matrix cores and the loads into LDS, which share the waves: 256 x 256 tiles
// take 128 bytes from L2 for 32 k of 4096 matrix cycles; alone the products of dx above take
// 383 us (1.43 PFLOP/s) and the loads 399, together 488.  Eight waves of 4 x 2
// fragments, two to a SIMD, since a wave that waits to issue a load issues no products: four
// of 4 x 4, with less LDS traffic, took 612.  Hence also the loads a few at a time between
// the products, a step's last fragments in registers before its barrier, and the next
// step's first ones read under the last products.
template <class E, bool ACOL, bool BCOL, bool GATED, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM * WN * kWave, 2) void product_kernel(Product<E> g) {
  constexpr int TK = tile_k(GATED), kStages = tile_stages(GATED);
  constexpr int THREADS = WM * WN * kWave, TM = WM * FM * 32, TN = WN * FN * 32;
  constexpr int NOUT = GATED ? TN / 2 : TN;  // output columns of a tile
  constexpr int HN = FN / 2;                 // gated: fragments of each kind
  static_assert(!GATED || (FN % 2 == 0 && !BCOL), "a wave holds gate and up columns");
  extern __shared__ __align__(16) uint16_t s_tiles[];  // kStages buffers of (A, B)
  constexpr int kA = TM * TK, kBuf = (TM + TN) * TK;
  const int w = wave_id(), wm = w / WN, wn = w % WN;

  // consecutive ids share an XCD; bands of 8 tile rows keep their operands in its L2
  const int total = static_cast<int>(gridDim.x), per = total / 8, bid = static_cast<int>(blockIdx.x);
  int id = bid < per * 8 ? (bid % 8) * per + bid / 8 : bid;
  const int tiles = g.tiles_m * g.tiles_n;
  const int split = id / tiles;
  id -= split * tiles;
  const int band = id / (8 * g.tiles_n), first = band * 8, in_band = min(8, g.tiles_m - first);
  const int m0 = (first + (id - band * 8 * g.tiles_n) % in_band) * TM;
  const int n0 = (id - band * 8 * g.tiles_n) / in_band * NOUT;

  const int k_tiles = max(1, (g.K + TK - 1) / TK);
  const int kt0 = split * g.per_split, kt1 = min(kt0 + g.per_split, k_tiles);
  const int steps = (kt1 - kt0) * g.parts * g.combos;

  TileLoad<ACOL, TM, TK, THREADS> load_a;
  TileLoad<BCOL, GATED ? TN / 2 : TN, TK, THREADS> load_b;
  load_a.init(g.a.ld, m0, g.M);
  load_b.init(g.b.ld, n0, g.N);
  // where the next tile's elements (m0, k) and (n0, k) are, and how much k is left of its
  // stretch (none past the last: zeros, unread)
  int next_kt = kt0, part = 0, combo = 0, left = 0;
  const uint16_t *pa, *pb[2];
  const auto stretch = [&] {
    const int k0 = next_kt * TK;
    left = combo < g.combos ? g.K - k0 : 0;
    // the last of them: (0,0); two: (1,0) before it
    const int c = combo >= g.combos || g.combos == 1 ? 5 : g.combos == 2 ? 3 + 2 * combo : combo;
    const long long qa = plane_a(c) * g.a.plane + (ACOL ? m0 + k0 * g.a.ld : m0 * g.a.ld + k0);
    const long long qb = plane_b(c) * g.b.plane + (BCOL ? n0 + k0 * g.b.ld : n0 * g.b.ld + k0);
    pa = g.a.p[part] + qa;
    pb[0] = g.b.p[GATED ? 0 : part] + qb;
    pb[1] = GATED ? g.b.p[1] + qb : nullptr;
  };
  stretch();
  const long long step_a = ACOL ? TK * g.a.ld : TK, step_b = BCOL ? TK * g.b.ld : TK;
  constexpr int kRa = decltype(load_a)::kRounds, kRb = decltype(load_b)::kRounds;
  constexpr int kLoads = kRa + (GATED ? 2 : 1) * kRb;
  // loads q0 .. q1 - 1 of the next tile; the tile after it once all are asked for
  const auto load = [&](int buf, int q0, int q1) {
    uint16_t* s = s_tiles + buf * kBuf;
#pragma unroll
    for (int q = q0; q < q1; ++q) {
      if (q < kRa) load_a.load(q, s, pa, left);
      else if (q < kRa + kRb) load_b.load(q - kRa, s + kA, pb[0], left);
      else load_b.load(q - kRa - kRb, s + kA + TN / 2 * TK, pb[1], left);
    }
  };
  const auto advance = [&] {
    if (++next_kt == kt1) {
      next_kt = kt0;
      if (++part == g.parts) { part = 0; ++combo; }
      stretch();
    } else {
      left -= TK;
      pa += step_a;
      pb[0] += step_b;
      if constexpr (GATED) pb[1] += step_b;
    }
  };
  bf16x8 fa[2][FM], fb[2][FN];
  const auto fragments = [&](int buf, int kk, int set) {
    const uint16_t* sa = s_tiles + buf * kBuf;
    const uint16_t* sb = sa + kA;
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[set][i] = load_frag<ACOL, TM, TK>(sa, wm * FM * 32 + i * 32, kk);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      if constexpr (GATED)  // two tiles of TN / 2 rows, one after the other
        fb[set][j] = load_frag<false, TN / 2, TK>(sb + (j / HN) * (TN / 2) * TK, wn * HN * 32 + (j % HN) * 32, kk);
      else
        fb[set][j] = load_frag<BCOL, TN, TK>(sb, wn * FN * 32 + j * 32, kk);
    }
  };

  floatx16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const auto products = [&](int set) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = mfma_bf16(fa[set][i], fb[set][j], acc[i][j]);
  };
  // how a stretch of the loop is laid out: a products' share after every read or load
  constexpr int kReads = (ACOL ? 2 : 1) * FM + (BCOL ? 2 : 1) * FN;  // LDS reads of a fragment set
  constexpr int kMfma = FM * FN;
  constexpr int kSteps = TK / 16;
  static_assert(kSteps % 2 == 0 && kLoads * (kStages - 1) < 64, "an even number of k steps; loads in flight are counted in 6 bits");
  // this wave's share of the oldest tile on its way has landed and its LDS reads so far
  // have come back, then everyone's
  const auto arrive = [&] {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads * (kStages - 2)) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  for (int i = 0; i + 1 < kStages; ++i) {
    load(i, 0, kLoads);
    advance();
  }
  arrive();
  // a tile's loads are spread over its predecessor's steps, the first after its barrier
  constexpr int kEarly = kLoads / kSteps;
  load(kStages - 1, 0, kEarly);
  fragments(0, 0, 0);
  int buf = 0, last = kStages - 1;  // the tile read, the one whose loads are partly asked for
  for (int step = 0; step < steps; ++step) {
    const int next = buf + 1 == kStages ? 0 : buf + 1;
#pragma unroll
    for (int kk = 0; kk < kSteps - 1; ++kk) {
      fragments(buf, kk + 1, (kk + 1) & 1);
      load(last, kEarly + kk * (kLoads - kEarly) / (kSteps - 1), kEarly + (kk + 1) * (kLoads - kEarly) / (kSteps - 1));
      __builtin_amdgcn_s_setprio(1);
      products(kk & 1);
      __builtin_amdgcn_s_setprio(0);
      interleave<0x100, kReads, kMfma / 2>();
      interleave<0x020, (kLoads - kEarly) / (kSteps - 1), kMfma - kMfma / 2>();
    }
    advance();
    arrive();
    fragments(next, 0, 0);
    load(buf, 0, kEarly);
    __builtin_amdgcn_s_setprio(1);
    products(1);
    __builtin_amdgcn_s_setprio(0);
    interleave<0x100, kReads, kMfma / 2>();
    interleave<0x020, kEarly, kMfma - kMfma / 2>();
    last = buf;
    buf = next;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is on its way into LDS at the end

  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), l32 = lane & 31, half = lane >> 5;
  if (!GATED || sizeof(E) == 4) {
    // the elements of a fragment that are not finite
    const int pla = g.combos == 6 ? 3 : g.combos, plb = g.combos == 6 ? 3 : 1;
    const int k_end = min(kt1 * TK, g.K);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const floatx16 one[1] = {acc[i][j]};
        if (g.combos > 1 && any_nonfinite(one)) {
          floatx16 c = {};
          for (int part = 0; part < g.parts; ++part)
#pragma unroll 1
            for (int k = kt0 * TK; k < k_end; k += 2) {
              const float va = element<ACOL>(g.a, pla, part, m0 + wm * FM * 32 + i * 32 + l32, g.M, k + half, k_end);
              const float vb = GATED ? element<BCOL>(g.b, plb, j / HN, n0 + wn * HN * 32 + (j % HN) * 32 + l32, g.N, k + half, k_end)
                                     : element<BCOL>(g.b, plb, part, n0 + wn * FN * 32 + j * 32 + l32, g.N, k + half, k_end);
              c = mfma32(va, vb, c);
            }
#pragma unroll
          for (int r = 0; r < 16; ++r)
            acc[i][j][r] = fabsf(acc[i][j][r]) <= 3.4028234663852886e38f ? acc[i][j][r] : c[r];
        }
      }
  }

  // register r of lane l: row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32
  if constexpr (GATED) {
    if (g.splits > 1) {  // gated_sum_kernel has the epilogue
#pragma unroll
      for (int q = 0; q < FN; ++q) {
        const int n = n0 + wn * HN * 32 + q % HN * 32 + l32;
        float* at = g.part + (split * 2 + q / HN) * (static_cast<size_t>(g.M) * g.N) + n;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int m = m0 + wm * FM * 32 + i * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
            if (n < g.N && m < g.M) at[static_cast<size_t>(m) * g.N] = acc[i][q][r];
          }
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < HN; ++j) {
      const int n = n0 + wn * HN * 32 + j * 32 + l32;
      const bool in = n < g.N;
      const float bg = in && g.bias[0] != nullptr ? to_f(g.bias[0][n]) : 0.f;
      const float bu = in && g.bias[1] != nullptr ? to_f(g.bias[1][n]) : 0.f;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = m0 + wm * FM * 32 + i * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
          const float a = acc[i][j][r] + bg, b = acc[i][j + HN][r] + bu;
          if (in && m < g.M) {
            const long long at = m * g.ldc + n;
            g.c[0][at] = from_f<E>(activation_of(g.act, a) * b);
            if (g.save[0] != nullptr) {
              // read by the backward, long after: past the caches (600 -> 540 us at [8192, 2048] -> 8192)
              __builtin_nontemporal_store(a, &g.save[0][at]);
              __builtin_nontemporal_store(b, &g.save[1][at]);
            }
          }
        }
    }
  } else {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = m0 + wm * FM * 32 + i * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
        if (m >= g.M) continue;
        const int second = m >= g.half ? 1 : 0, row = m - second * g.half;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int n = n0 + wn * FN * 32 + j * 32 + l32;
          if (n >= g.N) continue;
          if (g.splits > 1) g.part[(static_cast<size_t>(split) * g.M + m) * g.N + n] = acc[i][j][r];
          else if (row < g.half_rows && g.c[second] != nullptr) g.c[second][row * g.ldc + n] = from_f<E>(acc[i][j][r]);
        }
      }
  }
}

// The splits' sums, in order.
template <class E>
__global__ __launch_bounds__(256) void product_sum_kernel(Product<E> g) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, n = static_cast<long long>(g.M) * g.N;
  if (i >= n) return;
  const int m = static_cast<int>(i / g.N), col = static_cast<int>(i % g.N);
  const int second = m >= g.half ? 1 : 0, row = m - second * g.half;
  if (row >= g.half_rows || g.c[second] == nullptr) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < g.splits; ++k) s += g.part[k * n + i];
  g.c[second][row * g.ldc + col] = from_f<E>(s);
}

// The same of a gated product, and its epilogue.
template <class E>
__global__ __launch_bounds__(256) void gated_sum_kernel(Product<E> g) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, n = static_cast<long long>(g.M) * g.N;
  if (i >= n) return;
  const int col = static_cast<int>(i % g.N);
  float a = 0.f, b = 0.f;
#pragma unroll 8
  for (int k = 0; k < g.splits; ++k) {
    a += g.part[2 * k * n + i];
    b += g.part[(2 * k + 1) * n + i];
  }
  if (g.bias[0] != nullptr) a += to_f(g.bias[0][col]);
  if (g.bias[1] != nullptr) b += to_f(g.bias[1][col]);
  g.c[0][i] = from_f<E>(activation_of(g.act, a) * b);
  if (g.save[0] != nullptr) {
    g.save[0][i] = a;
    g.save[1][i] = b;
  }
}

// ---- few rows ---------------------------------------------------------------------
// Few rows of x, 16 NT to a workgroup: the weights' traffic is all there is (9.4 us for two of
// [5632, 2048] in bf16; 11 at 4 rows), so each is read once, straight into fragments, and
// none goes through LDS.  A workgroup takes 16 outputs of both projections.  Its waves share
// k in blocks of 128 bytes of a row, whole lines (where a lane read 128 bytes by itself,
// lines left the L1 between its loads: 118 us for 16 rows of float32, 28 now), ask for kAhead
// blocks together, and add their sums in LDS in a fixed order.  float32 takes the fp32
// matrix instruction: nothing to split, and its rate is above the memory's.
constexpr int kRowWaves = 8, kRowOut = 16;
typedef float floatx4 __attribute__((ext_vector_type(4)));

// 16 bytes of a row: an operand of a 16 x 16 product, lane l's row l % 16, its k the
// (l / 16)-th stretch of 16 bytes in 64.
template <class E>
struct Piece {
  static constexpr int kN = 16 / static_cast<int>(sizeof(E));
  E v[kN];
  __device__ __forceinline__ void load(const E* p) {
    struct __attribute__((packed, aligned(sizeof(E)))) Any { u32x4 q; };
    const u32x4 q = reinterpret_cast<const Any*>(p)->q;  // whatever its alignment
    __builtin_memcpy(v, &q, 16);
  }
  __device__ __forceinline__ void load_some(const E* row, int k, int n) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = k + i < n ? row[k + i] : E{};
  }
};
__device__ __forceinline__ floatx4 product16(const Piece<bf16_t>& a, const Piece<bf16_t>& b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 product16(const Piece<float>& a, const Piece<float>& b, floatx4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
  return c;
}

template <class E>
struct FewRows {
  const E* x;
  const E* w[2];
  const E* bias[2];
  E* y;
  float* save[2];
  long long ld_x, ld_w[2];
  int T, D, F, act;
};

template <class E, int NT>
__global__ __launch_bounds__(kRowWaves * kWave, 4) void few_rows_kernel(FewRows<E> g) {
  constexpr int kAhead = NT == 1 ? 4 : NT == 2 ? 2 : 1;
  constexpr int kPiece = Piece<E>::kN, kStep = 4 * kPiece, kBlockK = 2 * kStep;
  __shared__ float s_sum[kRowWaves][2][NT][16 * 16];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), w = wave_id(), l16 = lane & 15, part = lane >> 4;
  const int f0 = static_cast<int>(blockIdx.x) * kRowOut;
  const int t0 = static_cast<int>(blockIdx.y) * 16 * NT;
  const E* row_w[2];
  const E* row_x[NT];
#pragma unroll
  for (int j = 0; j < 2; ++j) row_w[j] = g.w[j] + min(f0 + l16, g.F - 1) * g.ld_w[j];
#pragma unroll
  for (int t = 0; t < NT; ++t) row_x[t] = g.x + min(t0 + t * 16 + l16, g.T - 1) * g.ld_x;
  floatx4 acc[2][NT] = {};
  const auto products = [&](const Piece<E> (&pw)[2], const Piece<E> (&px)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[j][t] = product16(px[t], pw[j], acc[j][t]);
  };
  const int whole = g.D / kBlockK;
  for (int b0 = w; b0 < whole; b0 += kRowWaves * kAhead) {
    Piece<E> fw[kAhead][2][2], fx[kAhead][2][NT];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int b = b0 + q * kRowWaves;
      if (b >= whole) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = b * kBlockK + i * kStep + part * kPiece;
#pragma unroll
        for (int j = 0; j < 2; ++j) fw[q][i][j].load(row_w[j] + k);
#pragma unroll
        for (int t = 0; t < NT; ++t) fx[q][i][t].load(row_x[t] + k);
      }
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (b0 + q * kRowWaves < whole) {
#pragma unroll
        for (int i = 0; i < 2; ++i) products(fw[q][i], fx[q][i]);
      }
  }
  if (w == whole % kRowWaves) {  // the rest, zeros past D
#pragma unroll 1
    for (int k0 = whole * kBlockK; k0 < g.D; k0 += kStep) {
      Piece<E> fw[2], fx[NT];
      const int k = k0 + part * kPiece;
#pragma unroll
      for (int j = 0; j < 2; ++j) fw[j].load_some(row_w[j], k, g.D);
#pragma unroll
      for (int t = 0; t < NT; ++t) fx[t].load_some(row_x[t], k, g.D);
      products(fw, fx);
    }
  }
  // a lane's output l % 16, its tokens 4 (l / 16) + r
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) s_sum[w][j][t][(4 * part + r) * 16 + l16] = acc[j][t][r];
  __syncthreads();
  // outputs fastest, so that neighbouring lanes store neighbouring values
  for (int i = threadIdx.x; i < NT * 16 * kRowOut; i += kRowWaves * kWave) {
    const int t = i / (16 * kRowOut), at_sum = i % (16 * kRowOut), token = t0 + i / kRowOut, n = f0 + i % kRowOut;
    if (token >= g.T || n >= g.F) continue;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int v = 0; v < kRowWaves; ++v) {
      a += s_sum[v][0][t][at_sum];
      b += s_sum[v][1][t][at_sum];
    }
    if (g.bias[0] != nullptr) a += to_f(g.bias[0][n]);
    if (g.bias[1] != nullptr) b += to_f(g.bias[1][n]);
    const long long at = static_cast<long long>(token) * g.F + n;
    g.y[at] = from_f<E>(activation_of(g.act, a) * b);
    if (g.save[0] != nullptr) {
      g.save[0][at] = a;
      g.save[1][at] = b;
    }
  }
}

// ---- operands as bf16 planes ---------------------------------------------------
// x as the nearest bf16s of it and of what they leave; what is not finite as (x, 0, 0).
__device__ __forceinline__ void split3(float x, uint16_t (&t)[3]) {
  t[0] = from_f<bf16_t>(x).bits;
  t[1] = t[2] = 0;
  if (!(fabsf(x) <= 3.4028234663852886e38f)) return;
  if ((t[0] & 0x7fff) == 0x7f80) t[0] -= 1;  // rounded past the largest bf16
  const float r = x - to_f(bf16_t{t[0]});
  t[1] = from_f<bf16_t>(r).bits;
  t[2] = from_f<bf16_t>(r - to_f(bf16_t{t[1]})).bits;
}

__device__ __forceinline__ void put8(uint16_t* dst, const uint16_t (&v)[8]) {
  u32x4 q;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = v[2 * i] | (static_cast<uint32_t>(v[2 * i + 1]) << 16);
  *reinterpret_cast<u32x4*>(dst) = q;
}

// Rows of C elements as 1 (bf16) or 3 (float32) planes of rows of Cp, zeros from C on; up to
// three matrices in a launch, each from its own workgroup on.
template <class E>
struct PackJobs {
  const E* src[3];
  uint16_t* dst[3];
  long long ld[3], plane[3], chunks[3];  // chunks of 8 in all
  int C[3], Cp[3];
  bool pairs[3];  // every pair of elements is aligned
  unsigned first[3];
  int n;
};

template <class E>
__global__ __launch_bounds__(256) void pack_kernel(PackJobs<E> g) {
  int job = 0;
#pragma unroll
  for (int i = 1; i < 3; ++i)
    if (i < g.n && blockIdx.x >= g.first[i]) job = i;
  const long long i = static_cast<long long>(blockIdx.x - g.first[job]) * 256 + threadIdx.x;
  if (i >= g.chunks[job]) return;
  const int C = g.C[job], Cp = g.Cp[job], row = Cp / 8;
  const long long r = i / row;
  const int c = static_cast<int>(i % row) * 8;
  const E* s = g.src[job] + r * g.ld[job] + c;
  E x[8];
  if (c + 8 <= C && g.pairs[job]) {
    struct alignas(2 * sizeof(E)) Pair { E v[2]; };
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const Pair q = *reinterpret_cast<const Pair*>(s + k);
      x[k] = q.v[0];
      x[k + 1] = q.v[1];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = c + k < C ? s[k] : E{};
  }
  uint16_t t[3][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint16_t v[3] = {0, 0, 0};
    if constexpr (sizeof(E) == 4) split3(x[k], v);
    else v[0] = x[k].bits;
#pragma unroll
    for (int j = 0; j < 3; ++j) t[j][k] = v[j];
  }
#pragma unroll
  for (int j = 0; j < (sizeof(E) == 4 ? 3 : 1); ++j) put8(g.dst[job] + j * g.plane[job] + r * Cp + c, t[j]);
}

// ---- da, db ----------------------------------------------------------------------
constexpr int kRowsPer = 4, kRowsPerSum = 16;  // rows of a thread: without and with the biases' sums

// Eight values that are not needed again: read past the caches, which the next kernel's
// operands need more (with half as many rows a thread, 190 -> 157 us at [8192, 8192]).
__device__ __forceinline__ void read8(const float* p, float (&v)[8]) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
  const f32x4 b = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void read8(const bf16_t* p, float (&v)[8]) {
  const u32x4 q = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(q[i]);
    v[2 * i + 1] = bf16_hi(q[i]);
  }
}

// da and db side by side, [T][2 Fp] (1 or 3 planes, 2 in bf16 where TWO), zeros from F on, and each thread's
// sums over its rows for the biases' gradients (in float32, before any rounding).  Bound by
// memory: 12 bytes read and 4 written an element in bf16.  VEC: F and every row are
// multiples of 16 bytes, and a thread's eight columns move in vectors.
template <class E, int ACT, bool VEC, bool TWO>
__global__ __launch_bounds__(256) void gate_grad_kernel(const E* __restrict__ go, long long ld_go,
                                                        const float* __restrict__ a, const float* __restrict__ b,
                                                        uint16_t* __restrict__ dab, long long plane,
                                                        float* __restrict__ sums, int T, int F, int Fp, int rows_per) {
  const int groups = Fp / 8;
  const long long gid = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int rb = static_cast<int>(gid / groups), f0 = static_cast<int>(gid % groups) * 8;
  if (rb >= (T + rows_per - 1) / rows_per) return;
  float sa[8], sb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sa[i] = sb[i] = 0.f;
#pragma unroll 2
  for (int r = rb * rows_per; r < min(T, (rb + 1) * rows_per); ++r) {
    const long long at = static_cast<long long>(r) * F + f0;
    const E* g = go + r * ld_go + f0;
    float xa[8], xb[8], xg[8];
    if constexpr (VEC) {
      read8(a + at, xa);
      read8(b + at, xb);
      read8(g, xg);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = f0 + i < F;
        xa[i] = in ? a[at + i] : 0.f;
        xb[i] = in ? b[at + i] : 0.f;
        xg[i] = in ? to_f(g[i]) : 0.f;  // da = db = 0
      }
    }
    uint16_t ta[3][8], tb[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const ActGrad d = activate<ACT>(xa[i]);
      const float ga = xg[i] * xb[i] * d.d, gb = xg[i] * d.f;
      sa[i] += ga;
      sb[i] += gb;
      uint16_t va[3] = {0, 0, 0}, vb[3] = {0, 0, 0};
      if constexpr (sizeof(E) == 4 || TWO) {
        split3(ga, va);
        split3(gb, vb);
      } else {
        va[0] = from_f<bf16_t>(ga).bits;
        vb[0] = from_f<bf16_t>(gb).bits;
      }
#pragma unroll
      for (int j = 0; j < 3; ++j) { ta[j][i] = va[j]; tb[j][i] = vb[j]; }
    }
#pragma unroll
    for (int j = 0; j < (sizeof(E) == 4 ? 3 : TWO ? 2 : 1); ++j) {
      uint16_t* dst = dab + j * plane + static_cast<long long>(r) * 2 * Fp + f0;
      put8(dst, ta[j]);
      put8(dst + Fp, tb[j]);
    }
  }
  if (sums != nullptr) {
    float* dst = sums + static_cast<long long>(rb) * 2 * Fp + f0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { dst[i] = sa[i]; dst[Fp + i] = sb[i]; }
  }
}

// Column sums of [rows][2 Fp] in a fixed order, kBiasRows rows a workgroup: 64 columns, 4
// lanes of rows each.  With more rows than that their sums go to `next` for another pass, else
// to the gradients.
constexpr int kBiasRows = 128;

template <class E>
__global__ __launch_bounds__(256) void bias_grad_kernel(const float* __restrict__ sums, int rows, int F, int Fp,
                                                        float* __restrict__ next, E* ga, E* gb) {
  __shared__ float s_p[4][kWave];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1), w = wave_id();
  const int c = static_cast<int>(blockIdx.x) * kWave + lane;
  const int r0 = static_cast<int>(blockIdx.y) * kBiasRows, r1 = min(rows, r0 + kBiasRows);
  float s = 0.f;
  if (c < 2 * Fp)
#pragma unroll 16
    for (int r = r0 + w; r < r1; r += 4) s += sums[static_cast<long long>(r) * 2 * Fp + c];
  s_p[w][lane] = s;
  __syncthreads();
  if (w != 0 || c >= 2 * Fp) return;
  s = ((s_p[0][lane] + s_p[1][lane]) + s_p[2][lane]) + s_p[3][lane];
  if (next != nullptr) {
    next[static_cast<long long>(blockIdx.y) * 2 * Fp + c] = s;
    return;
  }
  E* out = c < Fp ? ga : gb;
  const int f = c < Fp ? c : c - Fp;
  if (f < F && out != nullptr) out[f] = from_f<E>(s);
}

// ---- host ------------------------------------------------------------------------
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// Row-major matrices of one shape (one, or the gate's and the up weights) as the two
// parts of an operand: themselves where every row can be read in place, else planes in
// the workspace.
template <class E>
struct Source {
  const E* src[2];
  int64_t ld[2], rows, cols;
  int n;
  bool direct() const {
    bool ok = sizeof(E) == 2 && cols % 8 == 0;
    for (int i = 0; i < n; ++i) ok = ok && aligned16(src[i]) && ld[i] % 8 == 0 && ld[i] == ld[0];
    return ok;
  }
  int64_t plane() const { return up8(rows * up8(cols)); }
  int64_t elems() const { return direct() ? 0 : n * plane() * (sizeof(E) == 4 ? 3 : 1); }  // of bf16
};

// The operand that m makes, its planes (if it needs any) at ws, as more of `jobs`.
template <class E>
Operand operand(const Source<E>& m, uint16_t* ws, PackJobs<E>* jobs) {
  Operand o{};
  o.ld = m.ld[0];
  for (int i = 0; i < m.n; ++i) o.p[i] = reinterpret_cast<const uint16_t*>(m.src[i]);
  if (m.direct()) return o;
  const int64_t cp = up8(m.cols);
  o.ld = cp;
  o.plane = m.plane();
  for (int i = 0; i < m.n; ++i) {
    uint16_t* dst = ws + i * (m.elems() / m.n);
    o.p[i] = dst;
    const int j = jobs->n++;
    jobs->src[j] = m.src[i];
    jobs->dst[j] = dst;
    jobs->ld[j] = m.ld[i];
    jobs->plane[j] = o.plane;
    jobs->chunks[j] = m.rows * (cp / 8);
    jobs->pairs[j] = m.ld[i] % 2 == 0 && (reinterpret_cast<uintptr_t>(m.src[i]) & (2 * sizeof(E) - 1)) == 0;
    jobs->C[j] = static_cast<int>(m.cols);
    jobs->Cp[j] = static_cast<int>(cp);
  }
  return o;
}

template <class E>
int pack(PackJobs<E> jobs, hipStream_t st) {
  int64_t blocks = 0;
  for (int i = 0; i < jobs.n; ++i) {
    jobs.first[i] = static_cast<unsigned>(blocks);
    blocks += (jobs.chunks[i] + 255) / 256;
  }
  if (blocks == 0) return OSSM_OK;  // nothing to copy, or nothing in it
  if (int rc = check_grid("gated", blocks, 256)) return rc;
  hipLaunchKernelGGL(pack_kernel<E>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, jobs);
  return launch_check("pack_kernel");
}

template <class E, bool ACOL, bool BCOL, bool GATED, int WM, int WN, int FM, int FN>
int launch_tiled(Product<E> g, hipStream_t st) {
  constexpr int TM = WM * FM * 32, TN = WN * FN * 32;
  constexpr int lds = tile_stages(GATED) * (TM + TN) * tile_k(GATED) * 2;
  g.tiles_m = (g.M + TM - 1) / TM;
  g.tiles_n = (g.N + (GATED ? TN / 2 : TN) - 1) / (GATED ? TN / 2 : TN);
  const int64_t grid = static_cast<int64_t>(g.tiles_m) * g.tiles_n * g.splits;
  if (int rc = check_grid("gated", grid, WM * WN * kWave)) return rc;
  auto kern = product_kernel<E, ACOL, BCOL, GATED, WM, WN, FM, FN>;
  if (int rc = hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                         "hipFuncSetAttribute"))
    return rc;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(grid)), dim3(WM * WN * kWave), lds, st, g);
  if (int rc = launch_check("product_kernel")) return rc;
  if (g.splits > 1) {
    const int64_t n = static_cast<int64_t>(g.M) * g.N;
    hipLaunchKernelGGL((GATED ? gated_sum_kernel<E> : product_sum_kernel<E>), dim3(static_cast<unsigned>((n + 255) / 256)),
                       dim3(256), 0, st, g);
    return launch_check(GATED ? "gated_sum_kernel" : "product_sum_kernel");
  }
  return OSSM_OK;
}

int64_t tiles(int64_t m, int64_t n, int64_t tm, int64_t tn) { return ((m + tm - 1) / tm) * ((n + tn - 1) / tn); }

// How many ways the k of an [M, N] product of `k_tiles` tiles, each `combos` steps, is split:
// towards two workgroups a CU, none with fewer than 8 steps (dx of [25600, 128] from 2 x 512
// in float32, 200 tiles: two ways and their sum 96 us, unsplit in tiles half as high 129).
int choose_splits(int64_t m, int64_t n, int64_t k_tiles, int64_t combos, int64_t cus) {
  const int64_t t = std::max<int64_t>(1, tiles(m, n, 128, 128));  // an input without columns has none
  return static_cast<int>(std::max<int64_t>(1, std::min({2 * cus / t, k_tiles * combos / 8, k_tiles})));
}

// The same for a forward, where few tiles have much to add: [626, 1954] -> 86 in float32, 20
// tiles, 120 us unsplit and 30 split, [384, 3540] -> 562 242 and 54.  Splitting has to save 24
// steps, of about 0.4 us, to pay for the sums' launch and traffic: in bf16 2686 k of 45 tiles
// 41 and 30, but 1096 k 15.5 and 19.6, 2112 k of 245 tiles in two 30 and 37.
int forward_splits(int64_t m, int64_t n, int64_t k_tiles, int64_t combos, int64_t cus) {
  const int splits = choose_splits(m, n, k_tiles, combos, cus);
  const int64_t steps = k_tiles * combos;
  return steps - steps / splits >= 24 ? splits : 1;
}

template <class E, bool ACOL, bool BCOL, bool GATED>
int launch_product(Product<E> g, int64_t cus, hipStream_t st) {
  const int k_tiles = std::max(1, (g.K + tile_k(GATED) - 1) / tile_k(GATED));
  g.per_split = (k_tiles + g.splits - 1) / g.splits;
  g.splits = (k_tiles + g.per_split - 1) / g.per_split;
  // Eight waves and tiles of 256 where they fill three quarters of the CUs and pad no more than a
  // quarter beyond tiles of 128 (training [5255, 2518] -> 717 in float32, dx of 210 tiles, 1350 ->
  // 1024 us, [2128, 2524] -> 1906 488 -> 321; [25534, 289] -> 479 in bf16, dx's 289 columns padded to 512, 270 -> 290, so not there).
  const int64_t large = tiles(g.M, g.N, 256, GATED ? 128 : 256), small = tiles(g.M, g.N, 128, GATED ? 64 : 128);
  if (g.splits == 1 && large * 4 >= 3 * cus && large * 16 <= small * 5)
    return launch_tiled<E, ACOL, BCOL, GATED, 2, 4, 4, 2>(g, st);
  // too few tiles to give every CU one and half of them two: half as high ([1001, 1022] -> 2730 in
  // float32, 344 tiles: 97 -> 89 us; not from 384 on)
  if (g.splits == 1 && small * 2 < 3 * cus)
    return launch_tiled<E, ACOL, BCOL, GATED, 2, 2, 1, 2>(g, st);
  return launch_tiled<E, ACOL, BCOL, GATED, 2, 2, 2, 2>(g, st);
}

constexpr int kCombos(size_t e) { return e == 4 ? 6 : 1; }

int check_gated(const char* what, int dtype, int act, int64_t T, int64_t D, int64_t F, std::initializer_list<int64_t> d_strides) {
  const std::string w(what);
  if (dtype != OSSM_F32 && dtype != OSSM_BF16) return set_error(OSSM_ERR_INVALID_ARGUMENT, w + ": unknown dtype");
  if (act < 0 || act > OSSM_ACT_RELU) return set_error(OSSM_ERR_INVALID_ARGUMENT, w + ": unknown activation");
  if (T < 0 || D < 0 || F < 0) return set_error(OSSM_ERR_INVALID_ARGUMENT, w + ": negative size");
  for (int64_t ld : d_strides) {
    if (ld < D) return set_error(OSSM_ERR_INVALID_ARGUMENT, w + ": a row stride is below the row");
    if (ld > (1 << 20)) return set_error(OSSM_ERR_UNSUPPORTED, w + ": row strides up to 2^20");
  }
  if (T > (1 << 26) || D > (1 << 20) || F > (1 << 19) || T * std::max(D, F) > (int64_t(1) << 40))
    return set_error(OSSM_ERR_UNSUPPORTED, w + ": size exceeds launch limits");
  return OSSM_OK;
}

template <class E>
struct Gated {
  const E* x;
  const E* w[2];
  const E* bias[2];
  int64_t ld_x, ld_w[2], T, D, F;
  int act;
  Source<E> rows() const { return {{x, nullptr}, {ld_x, 0}, T, D, 1}; }
  Source<E> weights() const { return {{w[0], w[1]}, {ld_w[0], ld_w[1]}, F, D, 2}; }
};

// Whether few_rows_kernel takes a forward, by itself and by the products, us: 32 rows of
// [2048] -> 5632 in bf16 17 and 17, 64 25 and 18; where the operands would be packed first, 128
// of them in float32 94 and 99, 32 39 and 86, and of [1022] -> 2730 in bf16 15 and 24.  Small
// products leave the products' tiles few: [512] -> 2048 in float32 18 and 31 at 256 rows, 34
// and 39 at 512; in bf16 both are the call's own 11.
bool few(int64_t T, int64_t D, int64_t F, bool packed, int64_t small) {
  return T <= (packed ? 128 : 32) || (T <= 512 && T * D * F <= small);
}

template <class E>
int few_rows(const Gated<E>& p, E* y, float* a, float* b, hipStream_t st) {
  const FewRows<E> g{p.x, {p.w[0], p.w[1]}, {p.bias[0], p.bias[1]}, y, {a, b}, p.ld_x, {p.ld_w[0], p.ld_w[1]},
                     static_cast<int>(p.T), static_cast<int>(p.D), static_cast<int>(p.F), p.act};
  const dim3 grid(static_cast<unsigned>((p.F + kRowOut - 1) / kRowOut), static_cast<unsigned>((p.T + 63) / 64));
  hipLaunchKernelGGL((p.T <= 16 ? few_rows_kernel<E, 1> : p.T <= 32 ? few_rows_kernel<E, 2> : few_rows_kernel<E, 4>), grid,
                     dim3(kRowWaves * kWave), 0, st, g);
  return launch_check("few_rows_kernel");
}

template <class E>
int forward(const Gated<E>& p, E* y, float* a, float* b, StreamCall& call, hipStream_t st) {
  const Source<E> px = p.rows(), pw = p.weights();
  if (few(p.T, p.D, p.F, !px.direct() || !pw.direct(), int64_t(1) << (sizeof(E) == 4 ? 29 : 28)))
    return few_rows(p, y, a, b, st);
  const int64_t cus = std::max(1, device_cu_count(call.device()));
  const int combos = kCombos(sizeof(E)), splits = forward_splits(p.T, 2 * p.F, p.D / tile_k(true), combos, cus);
  // planes, then the splits' sums; a plane's rows are multiples of 16 bytes
  const size_t o_part = static_cast<size_t>(px.elems() + pw.elems()) * 2;
  const size_t bytes = o_part + (splits > 1 ? static_cast<size_t>(splits) * 2 * p.T * p.F * 4 : 0);
  void* ws = nullptr;
  if (bytes > 0)
    if (int rc = acquire_workspace(call, bytes, &ws)) return rc;
  Product<E> g{};
  uint16_t* q = static_cast<uint16_t*>(ws);
  PackJobs<E> jobs{};
  g.a = operand(px, q, &jobs);
  g.b = operand(pw, q + px.elems(), &jobs);
  if (int rc = pack(jobs, st)) return rc;
  g.M = static_cast<int>(p.T);
  g.N = static_cast<int>(p.F);
  g.K = static_cast<int>(p.D);
  g.parts = 1;
  g.splits = splits;
  g.combos = combos;
  g.part = reinterpret_cast<float*>(static_cast<char*>(ws) + o_part);
  g.c[0] = y;
  g.ldc = p.F;
  for (int i = 0; i < 2; ++i) g.bias[i] = p.bias[i];
  g.save[0] = a;
  g.save[1] = b;
  g.act = p.act;
  return launch_product<E, false, false, true>(g, cus, st);
}

// bfloat16: up to this many da the gradients take them as two terms.  Rounded to one, their
// errors average out over all of them and leave 1.41 times that of an exact sum rounded to
// bf16, but where some are much larger than others it is up to 1.53 times with 2^16 of them,
// 1.47 with 2^18 and 1.44 with 2^19 (relu, twelve draws); few products cost hardly more for it
// ([16, 2048] -> 5632 91 and 93 us), many twice as much.
constexpr int64_t kTwoPlanes = 1 << 18;

template <class E>
int backward(const Gated<E>& p, const E* go, int64_t ld_go, const float* a, const float* b, E* gx, E* const gw[2], E* const gb[2],
             StreamCall& call, hipStream_t st) {
  const Source<E> px = p.rows(), pw = p.weights();
  const bool two = sizeof(E) == 2 && p.T * p.F <= kTwoPlanes;
  const int64_t Fp = up8(p.F), planes = sizeof(E) == 4 ? 3 : two ? 2 : 1, combos = sizeof(E) == 4 ? 6 : planes;
  const int64_t cus = std::max(1, device_cu_count(call.device()));
  const bool want_w = gw[0] != nullptr || gw[1] != nullptr, want_b = gb[0] != nullptr || gb[1] != nullptr;
  const int rows_per = want_b ? kRowsPerSum : kRowsPer;
  const int64_t dab_plane = p.T * 2 * Fp, rbs = (p.T + rows_per - 1) / rows_per;
  const int sx = choose_splits(p.T, p.D, p.F / tile_k(false), combos, cus);
  const int sw = choose_splits(2 * Fp, p.D, p.T / tile_k(false), combos, cus);
  const int64_t part = std::max<int64_t>(gx != nullptr && sx > 1 ? sx * p.T * p.D : 0, want_w && sw > 1 ? sw * 2 * Fp * p.D : 0);
  // bytes; every start a multiple of 16
  size_t at = 0;
  const auto take = [&](int64_t bytes) { const size_t o = at; at += static_cast<size_t>((bytes + 255) / 256 * 256); return o; };
  const size_t o_dab = take(dab_plane * planes * 2), o_x = take(want_w ? px.elems() * 2 : 0);
  const size_t o_w = take(gx != nullptr ? pw.elems() * 2 : 0), o_part = take(part * 4);
  const size_t o_sums = take(want_b ? (rbs + (rbs + kBiasRows - 1) / kBiasRows) * 2 * Fp * 4 : 0);
  void* ws = nullptr;
  if (int rc = acquire_workspace(call, at, &ws)) return rc;
  char* base = static_cast<char*>(ws);
  uint16_t* dab = reinterpret_cast<uint16_t*>(base + o_dab);
  float* sums = want_b ? reinterpret_cast<float*>(base + o_sums) : nullptr;
  const int T = static_cast<int>(p.T), F = static_cast<int>(p.F), D = static_cast<int>(p.D), fp = static_cast<int>(Fp);
  const bool vec = F % 8 == 0 && aligned16(go) && aligned16(a) && aligned16(b) && ld_go * static_cast<int64_t>(sizeof(E)) % 16 == 0;
  const int64_t grad_groups = (rbs * (Fp / 8) + 255) / 256;
  if (int rc = check_grid("gated", grad_groups, 256)) return rc;
  const auto grads = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    auto kern = vec ? gate_grad_kernel<E, ACT, true, false> : gate_grad_kernel<E, ACT, false, false>;
    if constexpr (sizeof(E) == 2)
      if (two) kern = vec ? gate_grad_kernel<E, ACT, true, true> : gate_grad_kernel<E, ACT, false, true>;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(grad_groups)), dim3(256), 0, st, go, ld_go, a, b, dab,
                       static_cast<long long>(dab_plane), sums, T, F, fp, rows_per);
    return launch_check("gate_grad_kernel");
  };
  const auto by_act = [&] {
    switch (p.act) {
      case OSSM_ACT_SILU: return grads(std::integral_constant<int, OSSM_ACT_SILU>{});
      case OSSM_ACT_GELU: return grads(std::integral_constant<int, OSSM_ACT_GELU>{});
      case OSSM_ACT_GELU_TANH: return grads(std::integral_constant<int, OSSM_ACT_GELU_TANH>{});
      case OSSM_ACT_SIGMOID: return grads(std::integral_constant<int, OSSM_ACT_SIGMOID>{});
      default: return grads(std::integral_constant<int, OSSM_ACT_RELU>{});
    }
  };
  if (int rc = by_act()) return rc;
  if (want_b) {
    // the sums shrink 128 rows to one a pass; the passes alternate between two stretches
    float* from = sums;
    float* to = sums + rbs * 2 * Fp;
    for (int64_t rows = rbs;;) {
      const int64_t groups = (rows + kBiasRows - 1) / kBiasRows;
      hipLaunchKernelGGL(bias_grad_kernel<E>, dim3(static_cast<unsigned>((2 * Fp + kWave - 1) / kWave), static_cast<unsigned>(groups)),
                         dim3(256), 0, st, static_cast<const float*>(from), static_cast<int>(rows), F, fp,
                         groups > 1 ? to : nullptr, gb[0], gb[1]);
      if (int rc = launch_check("bias_grad_kernel")) return rc;
      if (groups == 1) break;
      std::swap(from, to);
      rows = groups;
    }
  }
  Product<E> g{};
  g.combos = static_cast<int>(combos);
  g.part = reinterpret_cast<float*>(base + o_part);
  g.a.p[0] = dab;
  g.a.p[1] = dab + Fp;
  g.a.plane = dab_plane;
  g.a.ld = 2 * Fp;
  g.N = D;
  g.ldc = p.D;
  PackJobs<E> jobs{};
  const Operand w_op = gx != nullptr ? operand(pw, reinterpret_cast<uint16_t*>(base + o_w), &jobs) : Operand{};
  const Operand x_op = want_w ? operand(px, reinterpret_cast<uint16_t*>(base + o_x), &jobs) : Operand{};
  if (int rc = pack(jobs, st)) return rc;
  if (gx != nullptr) {
    g.b = w_op;
    g.M = T;
    g.K = F;
    g.parts = 2;
    g.splits = sx;
    g.half = g.half_rows = T;
    g.c[0] = gx;
    if (int rc = launch_product<E, false, true, false>(g, cus, st)) return rc;
  }
  if (want_w) {
    g.b = x_op;
    g.M = 2 * fp;
    g.K = T;
    g.parts = 1;
    g.splits = sw;
    g.half = fp;
    g.half_rows = F;
    g.c[0] = gw[0];
    g.c[1] = gw[1];
    if (int rc = launch_product<E, true, true, false>(g, cus, st)) return rc;
  }
  return OSSM_OK;
}

__global__ __launch_bounds__(256) void gated_zero_kernel(uint16_t* p, int64_t n) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) p[i] = 0;
}

int zero(void* p, int64_t bytes, hipStream_t st) {
  if (p == nullptr || bytes == 0) return OSSM_OK;
  const int64_t n = bytes / 2, groups = std::min<int64_t>((n + 255) / 256, 1 << 16);
  hipLaunchKernelGGL(gated_zero_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, static_cast<uint16_t*>(p), n);
  return launch_check("gated_zero_kernel");
}

}  // namespace
}  // namespace ossm

using namespace ossm;

extern "C" {

int ossm_gated_forward(int dtype, const void* x, int64_t ld_x, const void* w_gate, int64_t ld_gate, const void* w_up,
                       int64_t ld_up, const void* b_gate, const void* b_up, int activation, void* y, float* a, float* b,
                       int64_t rows, int64_t d_in, int64_t d_out, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "gated_forward";
  if (int rc = check_gated(what, dtype, activation, rows, d_in, d_out, {ld_x, ld_gate, ld_up})) return rc;
  if (rows == 0 || d_out == 0) return OSSM_OK;
  if (!y || (d_in > 0 && (!x || !w_gate || !w_up)) || (a == nullptr) != (b == nullptr))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  StreamCall call(st);
  if (call.status()) return call.status();
  const auto run = [&](auto e) {
    using E = decltype(e);
    const auto in = [](const void* q) { return static_cast<const E*>(q); };
    const Gated<E> p{in(x), {in(w_gate), in(w_up)}, {in(b_gate), in(b_up)}, ld_x, {ld_gate, ld_up}, rows, d_in, d_out, activation};
    return forward(p, static_cast<E*>(y), a, b, call, st);
  };
  return dtype == OSSM_BF16 ? run(bf16_t{}) : run(0.f);
}

int ossm_gated_backward(int dtype, const void* grad_y, int64_t ld_grad, const void* x, int64_t ld_x, const void* w_gate,
                        int64_t ld_gate, const void* w_up, int64_t ld_up, int activation, const float* a, const float* b,
                        void* grad_x, void* grad_w_gate, void* grad_w_up, void* grad_b_gate, void* grad_b_up,
                        int64_t rows, int64_t d_in, int64_t d_out, ossm_stream_t stream_v) {
  clear_error();
  const char* what = "gated_backward";
  if (int rc = check_gated(what, dtype, activation, rows, d_in, d_out, {ld_x, ld_gate, ld_up})) return rc;
  if (rows > 0 && ld_grad < d_out)
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": a row stride is below the row");
  hipStream_t st = static_cast<hipStream_t>(stream_v);
  const int64_t e = dtype == OSSM_BF16 ? 2 : 4;
  if (rows == 0 || d_out == 0 || d_in == 0) {
    if (int rc = zero(grad_x, rows * d_in * e, st)) return rc;
    if (int rc = zero(grad_w_gate, d_out * d_in * e, st)) return rc;
    if (int rc = zero(grad_w_up, d_out * d_in * e, st)) return rc;
    if (rows == 0 || d_out == 0) {
      if (int rc = zero(grad_b_gate, d_out * e, st)) return rc;
      return zero(grad_b_up, d_out * e, st);
    }
    grad_x = grad_w_gate = grad_w_up = nullptr;
  }
  if (!grad_y || !a || !b || (d_in > 0 && (!x || !w_gate || !w_up)))
    return set_error(OSSM_ERR_INVALID_ARGUMENT, std::string(what) + ": null pointer");
  StreamCall call(st);
  if (call.status()) return call.status();
  const auto run = [&](auto t) {
    using E = decltype(t);
    const auto in = [](const void* q) { return static_cast<const E*>(q); };
    const auto out = [](void* q) { return static_cast<E*>(q); };
    const Gated<E> p{in(x), {in(w_gate), in(w_up)}, {nullptr, nullptr}, ld_x, {ld_gate, ld_up}, rows, d_in, d_out, activation};
    E* const gw[2] = {out(grad_w_gate), out(grad_w_up)};
    E* const gb[2] = {out(grad_b_gate), out(grad_b_up)};
    return backward(p, in(grad_y), ld_grad, a, b, out(grad_x), gw, gb, call, st);
  };
  return dtype == OSSM_BF16 ? run(bf16_t{}) : run(0.f);
}

}  // extern "C"
