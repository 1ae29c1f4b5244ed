// Log probabilities of given actions with the policy's entropy and its best alternatives, and the
// gradient of both with respect to the logits: pa_softmax_action_prob's softmax for action sets from
// a handful to a whole vocabulary, in logarithms, from fp32, bf16 or fp16 logits.  With z = l / T over
// the available actions, m = max z, s = sum exp(z - m):
//
//   log_prob = z_t - m - log s        entropy = log s - (1 / s) sum (z - m) exp(z - m)
//   dl_j = (1 / T) [ g_lp (delta_jt - p_j) - g_H p_j (log p_j + entropy) ]
//
// One pass: the running maximum and the two running sums are fp32 in every lane and are joined at the
// end (a sum s, u in front of maximum m becomes exp(m - m') s, exp(m - m') (u + (m - m') s) in front of
// m').  The alternatives are found in the same pass.  m, log s and the entropy are kept per row for the gradient,
// apart: the sum of the first two would round log s to the maximum's precision.
//
// Forward and gradient together move the logits three times and are bound by that: 4096 x 32768 bf16 in
// 163 us, 4.9 TB/s (forward 77 us while the gradient's 268 MB drain from the caches, gradient 87).
//
// An action is unavailable where the mask says so or its logit is -inf; whatever an unavailable
// place holds (NaN, +inf) is never used.  A row that leaves no action: log_prob -inf, entropy 0,
// alternatives -1, gradient 0.  A NaN or +inf among the available logits makes the row NaN.
#include <float.h>
#include <math.h>

#include "seq_common.hpp"

using namespace pa;
using namespace pa::seq;

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int MAX_TOP = 64;
// Distances from the maximum are clamped at -FLT_MAX, which stands for -inf and for all that is further: up
// to this temperature exp2(-FLT_MAX log2(e) / T) is zero (2^-184; at 1e38 it would be 0.03).
constexpr float MAX_TEMPERATURE = 0x1p121f;

template <typename T>
struct LpArgs {
  const T* logits; int64_t ld;
  int64_t rows; int A;
  const void* actions; int action_dtype;
  const uint8_t* mask; int64_t ldm;       // 1 = unavailable; or null; ldm 0: one row for all
  float inv_t;
  int top;
  float* log_prob; float* entropy; float* stats;   // stats [rows][3]: max logit, log s, entropy
  int64_t* top_actions; float* top_log_probs;      // [rows][top]
  int lane_shift;                          // small rows: log2 of the lanes per row
  int chunks; int64_t chunk;               // large rows: pieces of a row and their length
  float* part; uint64_t* part_keys;        // [rows][chunks][3], [rows][chunks][top]
  const float* g_lp; const float* g_h;     // [rows] or null
  T* d_logits;                             // [rows][A]
};

template <bool B>
struct Bool {
  static constexpr bool value = B;
};

// m, s, u of some of a row's elements, in units of the logits; empty: m = -inf, s = u = 0
struct Sums {
  float m, s, u;
};


// brings the sums in front of a new maximum
__device__ __forceinline__ void move_to(Sums& x, float m, float c) {
  if (x.s > 0.0f) {
    const float d = fmaxf(x.m - m, -FLT_MAX), f = __builtin_amdgcn_exp2f(d * c);
    x.u = f > 0.0f ? f * (x.u + d * x.s) : 0.0f;
    x.s *= f;
  }
  x.m = m;
}
__device__ __forceinline__ Sums join(Sums x, Sums y, float c) {
  const float m = __builtin_elementwise_maximum(x.m, y.m);
  move_to(x, m, c);
  move_to(y, m, c);
  return {m, x.s + y.s, x.u + y.u};
}
// of all lanes of a wave: the maximum first, so that every lane moves its sums once
__device__ __forceinline__ Sums join_lanes(Sums x, float c) {
  float m = x.m;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) m = __builtin_elementwise_maximum(m, __shfl_xor(m, o));
  move_to(x, m, c);
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    x.s += __shfl_xor(x.s, o);
    x.u += __shfl_xor(x.u, o);
  }
  return x;
}
// the elements' maximum must be taken first: e <= 1.  An element below the maximum by more than the
// range of a float, -inf among them, adds nothing.
__device__ __forceinline__ void add_to(Sums& x, float v, float c) {
  const float d = fmaxf(v - x.m, -FLT_MAX), e = __builtin_amdgcn_exp2f(d * c);
  x.s += e;
  x.u = fmaf(e, d, x.u);
}

// The same for N elements at once without the clamp, which costs an instruction an element: an -inf among
// them turns the second sum into NaN, and the elements are added again with it.
template <int N>
__device__ __forceinline__ void add_all(Sums& x, const float (&v)[N], float c) {
  float s = x.s, u = x.u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = v[i] - x.m, e = __builtin_amdgcn_exp2f(d * c);
    s += e;
    u = fmaf(e, d, u);
  }
  if (u == u) {
    x.s = s;
    x.u = u;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) add_to(x, v[i], c);
  }
}

// order of the alternatives: larger logits first, then lower index; NaN ranks above all.  0: none.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  if (v == -INFINITY) return 0;
  uint32_t u = __float_as_uint(v + 0.0f);
  u = (u >> 31) ? ~u : u | 0x80000000u;
  if (v != v) u = 0xffffffffu;
  return ((uint64_t)u << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  if (key == 0) return -INFINITY;
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u >> 31) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int from) {
  const uint32_t lo = __shfl((int)(uint32_t)v, from), hi = __shfl((int)(uint32_t)(v >> 32), from);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t xor_u64(uint64_t v, int o) {
  const uint32_t lo = __shfl_xor((int)(uint32_t)v, o), hi = __shfl_xor((int)(uint32_t)(v >> 32), o);
  return ((uint64_t)hi << 32) | lo;
}

template <typename T>
__device__ __forceinline__ int64_t action_of(const LpArgs<T>& a, int64_t row) {
  return a.action_dtype == PA_I64 ? reinterpret_cast<const int64_t*>(a.actions)[row]
                                  : (int64_t) reinterpret_cast<const int32_t*>(a.actions)[row];
}
template <typename T>
__device__ __forceinline__ float logit_of(const LpArgs<T>& a, int64_t row, int64_t j) {
  if (a.mask && a.mask[row * a.ldm + j]) return -INFINITY;
  return (float)a.logits[row * a.ld + j];
}

// log p of a logit below (or at) the maximum.  The distance is taken in halves: between the ends of the range it
// would pass it, where divided by T it need not.
__device__ __forceinline__ float log_prob_of(float v, float m, float inv_t, float log_s) {
  return (0.5f * v - 0.5f * m) * inv_t * 2.0f - log_s;
}

// one lane per row writes what the sums say
template <typename T>
__device__ __forceinline__ void finish_row(const LpArgs<T>& a, int64_t row, const Sums& x, float& log_s) {
  log_s = logf(x.s);
  const bool bad = x.m != x.m || x.m == INFINITY, none = x.m == -INFINITY;
  float h = none ? 0.0f : log_s - (x.u / x.s) * a.inv_t;
  if (bad) h = log_s = __builtin_nanf("");
  const int64_t t = action_of(a, row);
  float lp;
  if (t == -1) lp = 0.0f;
  else if (t < 0 || t >= a.A) lp = __builtin_nanf("");
  else {
    const float v = logit_of(a, row, t);
    lp = bad ? __builtin_nanf("") : v == -INFINITY ? -INFINITY : log_prob_of(v, x.m, a.inv_t, log_s);
  }
  a.log_prob[row] = lp;
  a.entropy[row] = h;
  if (a.stats) {
    a.stats[3 * row] = x.m;
    a.stats[3 * row + 1] = log_s;
    a.stats[3 * row + 2] = h;
  }
}
template <typename T>
__device__ __forceinline__ void write_top(const LpArgs<T>& a, int64_t row, int k, uint64_t key, const Sums& x,
                                          float log_s) {
  a.top_actions[row * a.top + k] = key ? (int64_t)(uint32_t)~(uint32_t)key : -1;
  a.top_log_probs[row * a.top + k] = key ? log_prob_of(value_of(key), x.m, a.inv_t, log_s) : -INFINITY;
}

// ---- up to 256 actions: a few lanes per row, four actions per lane, all in registers ---------------
// (65536 x 16 fp32 with masks: 5.3 us forwards, 6.2 backwards, 17 MB in all)
constexpr int SMALL = 256;

template <typename T>
__device__ __forceinline__ void load_four(const LpArgs<T>& a, int64_t row, int j, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = j + i < a.A ? logit_of(a, row, j + i) : -INFINITY;
}

template <typename T, bool TOP>
__global__ __launch_bounds__(256) void small_kernel(LpArgs<T> a) {
  const int lanes = 1 << a.lane_shift, rows = 256 >> a.lane_shift;
  const int lane = threadIdx.x & (lanes - 1);
  const float c = a.inv_t * LOG2E;
  for (int64_t r0 = (int64_t)blockIdx.x * rows; r0 < a.rows; r0 += (int64_t)gridDim.x * rows) {
    const int64_t mine = r0 + (threadIdx.x >> a.lane_shift);
    const bool on = mine < a.rows;
    const int64_t row = on ? mine : a.rows - 1;     // every lane takes part in the shuffles
    float f[4];
    load_four(a, row, lane * 4, f);
    Sums x = {__builtin_elementwise_maximum(__builtin_elementwise_maximum(f[0], f[1]), __builtin_elementwise_maximum(f[2], f[3])), 0.0f, 0.0f};
    for (int o = 1; o < lanes; o *= 2) x.m = __builtin_elementwise_maximum(x.m, __shfl_xor(x.m, o));
#pragma unroll
    for (int i = 0; i < 4; ++i) add_to(x, f[i], c);
    for (int o = 1; o < lanes; o *= 2) {
      x.s += __shfl_xor(x.s, o);
      x.u += __shfl_xor(x.u, o);
    }
    float log_s;
    if (on && lane == 0) finish_row(a, row, x, log_s);
    if constexpr (TOP) {
      log_s = (x.m != x.m || x.m == INFINITY) ? __builtin_nanf("") : logf(x.s);
      uint64_t key[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) key[i] = key_of(f[i], lane * 4 + i);
      for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) best = key[i] > best ? key[i] : best;
        for (int o = 1; o < lanes; o *= 2) {
          const uint64_t y = xor_u64(best, o);
          best = y > best ? y : best;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key[i] == best) key[i] = 0;
        if (on && lane == (k & (lanes - 1))) write_top(a, row, k, best, x, log_s);
      }
    }
  }
}

// ---- larger rows: waves stream a row or a piece of it ------------------------------------------------
// The best keys of a wave, sorted, one per lane.
struct Best {
  uint64_t key;
  // bitonic sequence over the lanes -> descending
  __device__ __forceinline__ void merge(int lane) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t y = xor_u64(key, o);
      key = ((lane & o) == 0) == (key > y) ? key : y;
    }
  }
  __device__ __forceinline__ void sort(int lane) {
#pragma unroll
    for (int n = 2; n <= 64; n *= 2)
#pragma unroll
      for (int o = n / 2; o > 0; o >>= 1) {
        const uint64_t y = xor_u64(key, o);
        const bool up = (lane & n) != 0 && n < 64;           // ascending blocks
        const bool first = (lane & o) == 0;
        key = (first != up) == (key > y) ? key : y;
      }
  }
  // `other` sorted the same way, in reverse lane order
  __device__ __forceinline__ void join_reversed(uint64_t other, int lane) {
    key = other > key ? other : key;
    merge(lane);
  }
  __device__ __forceinline__ void insert(uint64_t k, int lane) {
    const int at = __popcll(__ballot(key > k));
    const uint64_t before = shfl_u64(key, lane > 0 ? lane - 1 : 0);
    key = lane < at ? key : lane == at ? k : before;
  }
};

// What a lane reads at once: U packs of logits and their mask bytes.  A pack that would pass the end of
// the row is moved back to end with it, so that all are whole; what is not of this place is left out later.
template <typename T, int U>
struct Batch {
  static constexpr int V = 16 / (int)sizeof(T);
  Pack<T, V> p[U];
  uint32_t m[U][V / 4];
};
template <typename T, int U>
__device__ __forceinline__ void load_batch(Batch<T, U>& r, const T* src, const uint8_t* msk, int64_t j0, int step, int A) {
  constexpr int V = Batch<T, U>::V;
  typedef uint32_t B __attribute__((aligned(1), may_alias));
#pragma unroll
  for (int q = 0; q < U; ++q) {
    const int64_t j = j0 + (int64_t)q * step, at = j < A - V ? j : A - V;
    r.p[q] = load_pack<T, V>(src + at);
    if (msk)
#pragma unroll
      for (int k = 0; k < V / 4; ++k) r.m[q][k] = reinterpret_cast<const B*>(msk + at)[k];
  }
}

// W waves share a row's piece; 4 / W pieces per workgroup
template <typename T, int W, bool TOP>
__global__ __launch_bounds__(256) void large_kernel(LpArgs<T> a) {
  constexpr int V = 16 / (int)sizeof(T), U = 4;
  constexpr int STEP = W * 64 * V;
  __shared__ Sums sums[4];
  __shared__ uint64_t lists[TOP ? 4 : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part_wave = wave & (W - 1);
  const float c = a.inv_t * LOG2E;
  const int64_t pieces = a.rows * a.chunks;
  for (int64_t p0 = (int64_t)blockIdx.x * (4 / W); p0 < pieces; p0 += (int64_t)gridDim.x * (4 / W)) {
    const int64_t piece = p0 + wave / W;
    const bool on = piece < pieces;
    const int64_t row = on ? piece / a.chunks : 0, ch = on ? piece % a.chunks : 0;
    const int64_t j1 = !on ? 0 : (ch + 1) * a.chunk < a.A ? (ch + 1) * a.chunk : a.A;
    const T* src = a.logits + row * a.ld;
    const uint8_t* msk = a.mask ? a.mask + row * a.ldm : nullptr;
    Sums x = {-INFINITY, 0.0f, 0.0f};
    Best best = {0};
    uint64_t least = 0;            // the key that a new alternative has to pass
    float least_value = -INFINITY;
    bool seeded = false;
    int64_t base = ch * a.chunk + (int64_t)part_wave * 64 * V;
    constexpr int64_t BATCH = (int64_t)STEP * U;
    const auto sum_up = [&](const Batch<T, U>& cur) {
      float f[U][V];
#pragma unroll
      for (int q = 0; q < U; ++q) unpack<T, V>(cur.p[q], f[q]);
      if (msk) {
#pragma unroll
        for (int q = 0; q < U; ++q)
#pragma unroll
          for (int i = 0; i < V; ++i)
            if ((cur.m[q][i / 4] >> (8 * (i & 3))) & 0xff) f[q][i] = -INFINITY;
      }
      if (base + (int64_t)(U - 1) * STEP + 64 * V > j1) {       // some of the packs pass the end of the piece
#pragma unroll
        for (int q = 0; q < U; ++q) {
          const int64_t j = base + (int64_t)q * STEP + lane * V, at = j < a.A - V ? j : a.A - V;
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (at + i < j || at + i >= j1) f[q][i] = -INFINITY;
        }
      }
      float bm = f[0][0];      // maximum, not fmax: a NaN stays
#pragma unroll
      for (int q = 0; q < U; ++q)
#pragma unroll
        for (int i = 0; i < V; ++i) bm = __builtin_elementwise_maximum(bm, f[q][i]);
      if (!(bm <= x.m) && x.m == x.m) move_to(x, bm, c);
      if (msk) {
#pragma unroll
        for (int q = 0; q < U; ++q)
#pragma unroll
          for (int i = 0; i < V; ++i) add_to(x, f[q][i], c);
      } else {
#pragma unroll
        for (int q = 0; q < U; ++q) add_all<V>(x, f[q], c);
      }

      if constexpr (TOP) {
        uint64_t skip = 0;
        if (!seeded) {
          // the lanes' own best, sorted, are a first list: few others pass its k-th
#pragma unroll
          for (int q = 0; q < U; ++q)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const int64_t j = base + (int64_t)q * STEP + lane * V, at = j < a.A - V ? j : a.A - V;
              const uint64_t k = key_of(f[q][i], (uint32_t)(at + i));
              skip = k > skip ? k : skip;
            }
          best.key = skip;
          best.sort(lane);
          least = shfl_u64(best.key, a.top - 1);
          least_value = value_of(least);
          seeded = true;
        }
        if (__any(!(bm < least_value) && bm != -INFINITY)) {
          uint32_t cand = 0;
#pragma unroll
          for (int q = 0; q < U; ++q)
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (!(f[q][i] < least_value) && f[q][i] != -INFINITY) cand |= 1u << (q * V + i);
          while (__any(cand != 0)) {
            // every lane's next candidate; its value is read again rather than indexed in registers
            uint64_t k = 0;
            if (cand) {
              const int e = __ffs(cand) - 1;
              cand &= cand - 1;
              const int64_t j = base + (int64_t)(e / V) * STEP + lane * V, at = (j < a.A - V ? j : a.A - V) + e % V;
              k = key_of((float)src[at], (uint32_t)at);
              if (k == skip) k = 0;
            }
            uint64_t todo = __ballot(k > least);
            while (todo) {
              const int from = __ffsll((unsigned long long)todo) - 1;
              best.insert(shfl_u64(k, from), lane);
              least = shfl_u64(best.key, a.top - 1);
              todo &= todo - 1;
              todo &= __ballot(k > least);
            }
          }
          least_value = value_of(least);
        }
      }
    };
    // two batches in turn: while one is summed the next is under way, and none is copied
    Batch<T, U> even, odd;
    if (base < j1) load_batch(even, src, msk, base + lane * V, STEP, a.A);
    while (base < j1) {
      if (base + BATCH < j1) load_batch(odd, src, msk, base + BATCH + lane * V, STEP, a.A);
      sum_up(even);
      base += BATCH;
      if (base >= j1) break;
      if (base + BATCH < j1) load_batch(even, src, msk, base + BATCH + lane * V, STEP, a.A);
      sum_up(odd);
      base += BATCH;
    }
    x = join_lanes(x, c);
    if constexpr (W > 1) {
      if (lane == 0) sums[wave] = x;
      if constexpr (TOP) lists[wave][lane] = best.key;
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int w = 1; w < W; ++w) {
          x = join(x, sums[w], c);
          if constexpr (TOP) best.join_reversed(lists[w][63 - lane], lane);
        }
      }
    }
    if (on && part_wave == 0) {
      if (a.chunks == 1) {
        float log_s = 0.0f;
        if (lane == 0) finish_row(a, row, x, log_s);
        if constexpr (TOP) {
          log_s = __shfl(log_s, 0);
          if (lane < a.top) write_top(a, row, lane, best.key, x, log_s);
        }
      } else {
        if (lane == 0) {
          a.part[3 * piece] = x.m;
          a.part[3 * piece + 1] = x.s;
          a.part[3 * piece + 2] = x.u;
        }
        if constexpr (TOP)
          if (lane < a.top) a.part_keys[piece * a.top + lane] = best.key;
      }
    }
    if constexpr (W > 1) __syncthreads();
  }
}

template <typename T, bool TOP>
__global__ __launch_bounds__(256) void finish_kernel(LpArgs<T> a) {
  __shared__ uint64_t lists[TOP ? 4 : 1][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const float c = a.inv_t * LOG2E;
  Best best = {0};
  if constexpr (TOP) {
    for (int ch = wave; ch < a.chunks; ch += 4) {
      const int from = 63 - lane;
      const uint64_t k = from < a.top ? a.part_keys[(row * a.chunks + ch) * a.top + from] : 0;
      best.join_reversed(k, lane);
    }
    lists[wave][lane] = best.key;
    __syncthreads();
  }
  if (wave) return;
  Sums x = {-INFINITY, 0.0f, 0.0f};
  for (int ch = lane; ch < a.chunks; ch += 64) {
    const float* p = a.part + 3 * (row * a.chunks + ch);
    x = join(x, Sums{p[0], p[1], p[2]}, c);
  }
  x = join_lanes(x, c);
  float log_s = 0.0f;
  if (lane == 0) finish_row(a, row, x, log_s);
  if constexpr (TOP) {
#pragma unroll
    for (int w = 1; w < 4; ++w) best.join_reversed(lists[w][63 - lane], lane);
    log_s = __shfl(log_s, 0);
    if (lane < a.top) write_top(a, row, lane, best.key, x, log_s);
  }
}

// ---- gradient -----------------------------------------------------------------------------------------
struct RowGrad {
  float m, log2s, g_lp, g_h, h;
  int64_t t;        // the action that gets g_lp, or -1
  bool none;
};
template <typename T>
__device__ __forceinline__ RowGrad row_grad(const LpArgs<T>& a, int64_t row) {
  RowGrad r;
  r.m = a.stats[3 * row];
  r.log2s = a.stats[3 * row + 1] * LOG2E;
  r.h = a.stats[3 * row + 2];
  r.g_lp = a.g_lp ? a.g_lp[row] : 0.0f;
  r.g_h = a.g_h ? a.g_h[row] : 0.0f;
  r.none = r.m == -INFINITY;
  r.t = action_of(a, row);
  if (r.t == -1) {
    r.g_lp = 0.0f;
  } else if (r.t < 0 || r.t >= a.A) {
    r.g_lp = __builtin_nanf("");
    r.t = -1;
  } else if (logit_of(a, row, r.t) == -INFINITY) {   // log_prob is -inf whatever the logits are
    r.g_lp = 0.0f;
    r.t = -1;
  }
  return r;
}
// What a row's elements share: dl = p (k0 + k1 log2 p), k0 = -(g_lp + g_H H), k1 = -g_H ln 2, over T.  In an
// ordinary row everything is finite and k0, k1 hold the 1 / T already.
constexpr float LOWEST = -1.0e4f;      // of log2 p: keeps p log p at zero where p has underflowed
struct Factors {
  float k0, k1, top;      // top: what the action taken gets on top
};
__device__ __forceinline__ Factors factors_of(const RowGrad& r, float inv_t) {
  return {-fmaf(r.g_h, r.h, r.g_lp) * inv_t, -r.g_h * LN2 * inv_t, r.g_lp * inv_t};
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }
__device__ __forceinline__ bool ordinary(const RowGrad& r, float inv_t) {
  const Factors f = factors_of(r, inv_t);
  return finite(r.m) && finite(r.h) && finite(f.k0) && finite(f.k1 * LOWEST) && finite(f.top);
}
// f: logits in (-inf: unavailable), gradients out.
// CHECK: the row is not an ordinary one (no action left, NaN, or a factor that has no end): nothing of that
// reaches unavailable places, and the division by T comes last, so that p = 0 gives 0 where only g / T passes
// the range of a float.
template <int N, bool CHECK>
__device__ __forceinline__ void grad_of(float (&f)[N], int64_t j, const RowGrad& r, float c, float inv_t) {
  const float by = CHECK ? 1.0f : inv_t;
  const Factors k = factors_of(r, by);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t2 = fmaxf(fmaf(f[i] - r.m, c, -r.log2s), LOWEST), p = __builtin_amdgcn_exp2f(t2);
    const float d = p * fmaf(k.k1, CHECK && p == 0.0f ? 1.0f : t2, k.k0);
    f[i] = CHECK && (f[i] == -INFINITY || r.none) ? 0.0f : d;
  }
  if (r.t >= j && r.t < j + N) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (j + i == r.t) f[i] = fmaf(r.g_lp, by, f[i]);
  }
  if constexpr (CHECK) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] *= inv_t;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void small_grad_kernel(LpArgs<T> a) {
  const int lanes = 1 << a.lane_shift, rows = 256 >> a.lane_shift;
  const int j = (threadIdx.x & (lanes - 1)) * 4;
  const float c = a.inv_t * LOG2E;
  for (int64_t row = (int64_t)blockIdx.x * rows + (threadIdx.x >> a.lane_shift); row < a.rows;
       row += (int64_t)gridDim.x * rows) {
    const RowGrad r = row_grad(a, row);
    float f[4];
    load_four(a, row, j, f);
    grad_of<4, true>(f, j, r, c, a.inv_t);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < a.A) a.d_logits[row * a.A + j + i] = (T)f[i];
  }
}

template <typename T>
__global__ __launch_bounds__(256) void large_grad_kernel(LpArgs<T> a) {
  constexpr int V = 16 / (int)sizeof(T), U = 4, STEP = 256 * V;
  const float c = a.inv_t * LOG2E;
  const int64_t per_row = (a.A + STEP * U - 1) / (STEP * U), pieces = a.rows * per_row;
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    const int64_t row = piece / per_row;
    const int64_t base = (piece - row * per_row) * STEP * U + threadIdx.x * V;
    const T* src = a.logits + row * a.ld;
    const uint8_t* msk = a.mask ? a.mask + row * a.ldm : nullptr;
    T* dst = a.d_logits + row * a.A;
    Batch<T, U> in;                     // a row's last pack is moved back; its places are written twice, alike
    load_batch(in, src, msk, base, STEP, a.A);
    const RowGrad r = row_grad(a, row);
    const auto write = [&](auto checked) {
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int64_t j = base + q * STEP, at = j < a.A - V ? j : a.A - V;
        float f[V];
        unpack<T, V>(in.p[q], f);
        if (msk) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if ((in.m[q][i / 4] >> (8 * (i & 3))) & 0xff) f[i] = -INFINITY;
        }
        grad_of<V, decltype(checked)::value>(f, at, r, c, a.inv_t);
        if (j < a.A) store_pack<T, V>(dst + at, pack<T, V>(f));
      }
    };
    if (ordinary(r, a.inv_t)) write(Bool<false>());
    else write(Bool<true>());
  }
}

// A row of up to this many batches of four waves is not cut: the launch that joins costs more than the
// batches do one after another (3 x 31698 bf16, a call: 12.9 us whole, 17.0 in four pieces; 300 rows with 20
// alternatives 23 and 33; 3 rows with 20 alternatives 21.2 and 19.9).
constexpr int WHOLE = 4;

// pieces of a row: few rows are cut so that the card is filled (16 x 131072 bf16 with 20 alternatives: 12.3
// us in 256 pieces and 6 us to join them; a row is 16 batches of a workgroup, about 2 us each, in one piece)
struct Pieces {
  int chunks;
  int64_t chunk, bytes, keys;
};
Pieces pieces_of(int64_t rows, int64_t A, int dtype, int top) {
  Pieces p = {1, A, 0, 0};
  const int64_t step = 4 * 256 * 16 / elem_size(dtype);    // what four waves read at once
  if (A > WHOLE * step && rows < 512) {
    int64_t chunks = ceil_div(1024, rows > 0 ? rows : 1);
    if (chunks > ceil_div(A, step)) chunks = ceil_div(A, step);
    if (chunks > 128) chunks = 128;
    p.chunk = round_up(ceil_div(A, chunks), step);
    p.chunks = (int)ceil_div(A, p.chunk);
  }
  if (p.chunks > 1) {
    p.keys = round_up(rows * p.chunks * 12, 256);
    p.bytes = p.keys + rows * p.chunks * top * 8;
  }
  return p;
}

unsigned grid_of(int64_t blocks) { return (unsigned)(blocks < (1 << 22) ? blocks : (1 << 22)); }

int lane_shift_of(int A) {
  int s = 0;
  while ((4 << s) < A) ++s;
  return s;
}

template <typename T>
LpArgs<T> args_of(const pa_log_probs_args* p) {
  LpArgs<T> a;
  memset(&a, 0, sizeof(a));
  a.logits = reinterpret_cast<const T*>(p->logits); a.ld = p->ld; a.rows = p->rows; a.A = p->A;
  a.actions = p->actions; a.action_dtype = p->action_dtype;
  a.mask = p->mask; a.ldm = p->ldm;
  a.inv_t = (float)(1.0 / (double)p->temperature);
  a.top = p->top; a.log_prob = p->log_prob; a.entropy = p->entropy; a.stats = p->stats;
  a.top_actions = p->top_actions; a.top_log_probs = p->top_log_probs;
  a.lane_shift = p->A <= SMALL ? lane_shift_of(p->A) : 0;
  a.g_lp = p->d_log_prob; a.g_h = p->d_entropy; a.d_logits = reinterpret_cast<T*>(p->d_logits);
  return a;
}

template <typename T, bool TOP>
int run_forward(const pa_log_probs_args* p, hipStream_t s) {
  LpArgs<T> a = args_of<T>(p);
  if (a.A <= SMALL) {
    hipLaunchKernelGGL((small_kernel<T, TOP>), dim3(grid_of(ceil_div(a.rows, 256 >> a.lane_shift))), dim3(256),
                       0, s, a);
    PA_LAUNCH_CHECK();
    return PA_OK;
  }
  const Pieces c = pieces_of(a.rows, a.A, p->dtype, a.top);
  a.chunks = c.chunks; a.chunk = c.chunk;
  a.part = reinterpret_cast<float*>(p->scratch);
  a.part_keys = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(p->scratch) + c.keys);
  if (a.A <= 4096) {
    hipLaunchKernelGGL((large_kernel<T, 1, TOP>), dim3(grid_of(ceil_div(a.rows * a.chunks, 4))), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((large_kernel<T, 4, TOP>), dim3(grid_of(a.rows * a.chunks)), dim3(256), 0, s, a);
  }
  PA_LAUNCH_CHECK();
  if (a.chunks > 1) {
    hipLaunchKernelGGL((finish_kernel<T, TOP>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    PA_LAUNCH_CHECK();
  }
  return PA_OK;
}

template <typename T>
int run_backward(const pa_log_probs_args* p, hipStream_t s) {
  const LpArgs<T> a = args_of<T>(p);
  if (a.A <= SMALL) {
    hipLaunchKernelGGL((small_grad_kernel<T>), dim3(grid_of(ceil_div(a.rows, 256 >> a.lane_shift))), dim3(256), 0,
                       s, a);
  } else {
    constexpr int PIECE = 256 * (16 / (int)sizeof(T)) * 4;
    hipLaunchKernelGGL((large_grad_kernel<T>), dim3(grid_of(a.rows * ceil_div(a.A, PIECE))), dim3(256), 0, s, a);
  }
  PA_LAUNCH_CHECK();
  return PA_OK;
}

int check_args(const char* who, const pa_log_probs_args* p) {
  PA_REQUIRE(p, PA_ERR_INVALID, "%s: null argument", who);
  PA_REQUIRE(elem_size(p->dtype), PA_ERR_UNSUPPORTED, "%s: logits dtype %d", who, p->dtype);
  PA_REQUIRE(p->action_dtype == PA_I64 || p->action_dtype == PA_I32, PA_ERR_UNSUPPORTED, "%s: action dtype %d", who,
             p->action_dtype);
  PA_REQUIRE(p->rows >= 0 && p->rows <= 0x7fffffffll && p->A >= 1 && p->ld >= 0 && p->ldm >= 0, PA_ERR_INVALID,
             "%s: bad shape (rows %lld, actions %d)", who, (long long)p->rows, p->A);
  PA_REQUIRE(p->temperature >= FLT_MIN && p->temperature <= MAX_TEMPERATURE, PA_ERR_INVALID,
             "%s: temperature %g (2^-126 to 2^121)", who, (double)p->temperature);
  PA_REQUIRE(p->rows == 0 || (p->logits && p->actions), PA_ERR_INVALID, "%s: null pointer", who);
  return PA_OK;
}

}  // namespace

extern "C" int64_t pa_action_log_probs_scratch(int64_t rows, int32_t A, int32_t dtype, int32_t top) {
  return rows <= 0 || A <= 0 || !elem_size(dtype) ? 0 : pieces_of(rows, A, dtype, top).bytes;
}

extern "C" int pa_action_log_probs(const pa_log_probs_args* args, void* stream) {
  const int rc = check_args("pa_action_log_probs", args);
  if (rc != PA_OK) return rc;
  PA_REQUIRE(args->top >= 0 && args->top <= MAX_TOP, PA_ERR_UNSUPPORTED, "pa_action_log_probs: top %d (0 to %d)",
             args->top, MAX_TOP);
  if (args->rows == 0) return PA_OK;
  PA_REQUIRE(args->log_prob && args->entropy && (args->top == 0 || (args->top_actions && args->top_log_probs)),
             PA_ERR_INVALID, "pa_action_log_probs: null output");
  PA_REQUIRE(args->scratch || pieces_of(args->rows, args->A, args->dtype, args->top).bytes == 0, PA_ERR_INVALID,
             "pa_action_log_probs: this shape needs scratch (pa_action_log_probs_scratch)");
  PA_ON_DEVICE(args->device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (args->dtype == PA_F32) return args->top ? run_forward<float, true>(args, s) : run_forward<float, false>(args, s);
  if (args->dtype == PA_BF16)
    return args->top ? run_forward<bf16_t, true>(args, s) : run_forward<bf16_t, false>(args, s);
  return args->top ? run_forward<f16_t, true>(args, s) : run_forward<f16_t, false>(args, s);
}

extern "C" int pa_action_log_probs_grad(const pa_log_probs_args* args, void* stream) {
  const int rc = check_args("pa_action_log_probs_grad", args);
  if (rc != PA_OK) return rc;
  if (args->rows == 0) return PA_OK;
  PA_REQUIRE(args->stats && args->d_logits, PA_ERR_INVALID, "pa_action_log_probs_grad: null pointer (stats, d_logits)");
  PA_ON_DEVICE(args->device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (args->dtype == PA_F32) return run_backward<float>(args, s);
  if (args->dtype == PA_BF16) return run_backward<bf16_t>(args, s);
  return run_backward<f16_t>(args, s);
}
