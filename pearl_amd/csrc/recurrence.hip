// Gated linear recurrence over a history and its backward pass; the many-channel, 16-bit,
// differentiable sibling of pa_ppo_gae's scalar recurrence.  Per batch row and channel
//
//   decay gates:  h_t = g_t h_{t-1} + x_t
//   logit gates:  h_t = a_t h_{t-1} + (1 - a_t) x_t,   a_t = 1 / (1 + exp(-g_t))
//
// An affine step h -> A h + H composes as (A2, H2) o (A1, H1) = (A2 A1, A2 H1 + H2), so a history is
// scanned in parallel.  A reset makes its step ignore the state before it: not a factor of zero (zero
// times infinity is not zero) but a flag that travels with the pair and selects.
//
// A workgroup owns a slab of 64 channels (a 128-byte line of 16-bit values) and walks the steps in tiles:
// 32 lanes of two channels side by side in a row, two groups of 8 consecutive steps per wave, waves behind
// one another in time.  Each lane scans its own steps, the groups are joined by one lane shuffle, the
// waves through LDS by one wave, which carries the state on, while the next tile's loads are already under
// way.  Every output is written once and every input read once, but for a workgroup's last prefetch, which finds
// no further tile and loads the last one again (a gradient without d_h loads rows of x in its place).  The state
// is fp32 throughout; only the stored h is rounded to the input's type.
//
// Two channels a lane, because what a step costs beside its loads is the joining: with eight a lane (16-byte
// loads) the tile needs three shuffles of 16 values (61 us against 49 at 16 x 2048 x 1024 bf16, 201 MB, which a
// copy moves in 39).  Forwards 21 VALU instructions a value, backwards 40; the rest of the time is the tile's
// two barriers.
//
// Where batch x channels give too few workgroups, the steps are cut into chunks: a first launch
// composes each chunk's pair, the second starts every chunk from the composition of those before it
// (1 x 65536 x 512 bf16: 30 + 40 us; the inputs are read twice).
//
// Backward, with G_t = dh_t + c_t and c_{t-1} = a_t G_t (0 at a reset), c_T = d_last:
//   decay:  dx = G, dg = G h_{t-1};   logit:  dx = (1 - a) G, dg = a (1 - a) G (h_{t-1} - x);
//   d_h0 = c_0.  The forward pass keeps the fp32 state in front of every 128th step;
// the states inside a tile are computed again from it rather than read back rounded.
#include "seq_common.hpp"

using namespace pa;
using namespace pa::seq;

namespace {

// A kernel's shape: NW waves, CL lanes side by side in a row (so 64 / CL groups of steps per wave), L
// consecutive steps per lane, V channels per lane.
template <int NW_, int CL_, int L_, int V_>
struct Shape {
  static constexpr int NW = NW_, CL = CL_, L = L_, V = V_, TG = 64 / CL_, STEPS = NW_ * TG * L_, SLAB = CL_ * V_;
};
typedef Shape<1, 16, 8, 2> Short;          // histories of up to 32 steps
typedef Shape<8, 16, 4, 2> Middle;         // of up to 128: half-width slabs (1 x 128 x 4096 fp32 6.2 us; as Long 14.4)
typedef Shape<16, 32, 8, 2> Long;          // longer ones, forwards
typedef Shape<8, 32, 8, 2> LongGrad;       // longer ones, backwards: 16 waves of 8 steps would spill (240 us, not 85)
constexpr int KEEP = Long::STEPS / LongGrad::STEPS;
static_assert(Short::SLAB <= 64 && Middle::SLAB <= 64 && Long::SLAB <= 64 && LongGrad::SLAB == Long::SLAB,
              "a lane of a wave carries the state of each channel");
static_assert(Long::STEPS % LongGrad::STEPS == 0 && Long::NW % KEEP == 0, "states are kept in front of waves");

template <typename T, typename G>
struct RecArgs {
  const T* x; int64_t x_b, x_t;
  const G* g; int64_t g_b, g_t;
  const float* h0;                               // [B][D] or null: zeros
  const uint8_t* resets; int64_t r_b, r_t;       // or null
  const int32_t* lengths;                        // [B] or null: T
  int64_t B, T_; int D;
  int reverse;
  int slabs, chunks; int64_t chunk_tiles, tiles;
  int64_t kept;                                  // states kept per history: the gradient's tiles
  float* agg_a; float* agg_h; uint8_t* agg_r;    // [B][chunks][D], [B][chunks] (decays: and [slabs]): the chunks' pairs
  T* h; float* last; float* carries;             // [B][T][D], [B][D] or null, [B][tiles][D] or null
  const T* dh; int64_t dh_b, dh_t;               // or null: zeros
  const float* d_last;                           // [B][D] or null
  T* dx; G* dg; float* dh0;                      // dh0 or null
};

// a and 1 - a of a logit, each to its own size also where it is tiny: the smaller is off by up to about
// (|z| + 4) 2^-24 of itself (the exponential's argument is rounded once), the larger by a few 2^-24.  Below -87
// a stays at 1.6e-38: a little further down the exponential would be infinite, and 1 - a infinity times zero.
// NaN stays NaN (maximum, not fmax).
__device__ __forceinline__ float exp_minus(float z) {
  return __builtin_amdgcn_exp2f(-1.44269504088896340736f * __builtin_elementwise_maximum(z, -87.0f));
}
__device__ __forceinline__ void gate_of(float e, float& a, float& keep) {
  a = __builtin_amdgcn_rcpf(1.0f + e);
  keep = e * a;
}

template <typename T, typename G, typename S>
struct Tile {
  Pack<T, S::V> x[S::L];
  Pack<G, S::V> g[S::L];
  uint32_t resets[S::L / 4];   // a byte per step
};

// The rows of one tile of a history of n steps.  Its step j lies in row first + j, or, read backwards,
// in row first + here - 1 - j.  A tile behind the end gets one row that exists, for its loads.
struct Rows {
  int64_t first;
  int here;        // steps of the tile that lie inside the history, at least 1
  int valid;       // the same, or 0
};
template <typename S>
__device__ __forceinline__ Rows rows_of(int64_t tile, int64_t n, int reverse) {
  const int64_t valid = n - tile * S::STEPS;
  Rows r;
  r.valid = valid <= 0 ? 0 : valid < S::STEPS ? (int)valid : S::STEPS;
  r.here = r.valid ? r.valid : 1;
  r.first = r.valid ? reverse ? valid - r.here : tile * S::STEPS : 0;
  return r;
}
// byte offset of step j within the tile's rows; steps behind the end fall on the last row.  Row strides
// are below 2^23 bytes, so one 24-bit multiply-add forms it and 31 bits hold it.
__device__ __forceinline__ uint32_t row_offset(int j, const Rows& r, int reverse, uint32_t stride, uint32_t at) {
  const int k = j < r.here ? j : r.here - 1;
  return __umul24(reverse ? r.here - 1 - k : k, stride) + at;
}
// In a full tile a lane's i-th row is the same distance from its first in every lane: `lane_rows` is the
// lane's part of its address, in rows, and step_row(i) the uniform part.  Accesses go through buffer
// descriptors, which take the uniform part in a scalar register and the lane's as one 32-bit offset:
// pointers would hold two vector registers and an addition for every row in flight.
template <typename S>
__device__ __forceinline__ int lane_rows(int j, int reverse) {
  return reverse ? S::STEPS - S::L - j : j;
}
template <typename S>
__device__ __forceinline__ int step_row(int i, int reverse) {
  return reverse ? S::L - 1 - i : i;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, 0x7ffffff0, 0x00020000);
}
template <typename T, int V, bool TINY>
__device__ __forceinline__ Pack<T, V> buffer_load(__amdgpu_buffer_rsrc_t b, uint32_t lane, uint32_t row) {
  Pack<T, V> p;
  if constexpr (TINY) {      // rows of one element
#pragma unroll
    for (int k = 0; k < Pack<T, V>::WORDS; ++k) p.w[k] = 0;
    p.w[0] = sizeof(T) == 4 ? __builtin_amdgcn_raw_buffer_load_b32(b, lane, row, 0)
                            : __builtin_amdgcn_raw_buffer_load_b16(b, lane, row, 0);
  } else if constexpr (Pack<T, V>::WORDS == 1) {
    p.w[0] = __builtin_amdgcn_raw_buffer_load_b32(b, lane, row, 0);
  } else {
    static_assert(Pack<T, V>::WORDS == 2, "two channels per lane");
    const auto u = __builtin_amdgcn_raw_buffer_load_b64(b, lane, row, 0);
    p.w[0] = u[0];
    p.w[1] = u[1];
  }
  return p;
}
template <typename T, int V, bool TINY>
__device__ __forceinline__ void buffer_store(__amdgpu_buffer_rsrc_t b, uint32_t lane, uint32_t row, const Pack<T, V>& p) {
  if constexpr (TINY) {
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(p.w[0], b, lane, row, 0);
    else __builtin_amdgcn_raw_buffer_store_b16((uint16_t)p.w[0], b, lane, row, 0);
  } else if constexpr (Pack<T, V>::WORDS == 1) {
    __builtin_amdgcn_raw_buffer_store_b32(p.w[0], b, lane, row, 0);
  } else {
    typedef uint32_t U __attribute__((ext_vector_type(2)));
    U u;
    u.x = p.w[0];
    u.y = p.w[1];
    __builtin_amdgcn_raw_buffer_store_b64(u, b, lane, row, 0);
  }
}

// The L rows of this lane from step j of the tile on, `c` channels into the row.  No branches between
// them, so that a tile's loads all go out at once; the selects on the step ignore what does not belong.
template <typename S, typename T, bool TINY>
__device__ __forceinline__ void load_rows(Pack<T, S::V> (&p)[S::L], const T* base, int64_t stride, int j, const Rows& r,
                                          int reverse, int c) {
  constexpr int V = S::V, L = S::L;
  const uint32_t step = (uint32_t)(stride * sizeof(T)), at = (uint32_t)(c * sizeof(T));
  const __amdgpu_buffer_rsrc_t rows = buffer_at(base + r.first * stride);
  if (r.valid == S::STEPS) {
    const uint32_t off = __umul24(lane_rows<S>(j, reverse), step) + at;
#pragma unroll
    for (int i = 0; i < L; ++i) p[i] = buffer_load<T, V, TINY>(rows, off, step * step_row<S>(i, reverse));
  } else {
#pragma unroll
    for (int i = 0; i < L; ++i) p[i] = buffer_load<T, V, TINY>(rows, row_offset(j + i, r, reverse, step, at), 0);
  }
}

// A byte for each of the lane's steps, in the order of the steps.
template <typename S, typename T, typename G>
__device__ __forceinline__ void load_resets(uint32_t (&p)[S::L / 4], const RecArgs<T, G>& a, int64_t b, int j,
                                            const Rows& r) {
  if (!a.resets) {
#pragma unroll
    for (int k = 0; k < S::L / 4; ++k) p[k] = 0;
    return;
  }
  const uint8_t* first = a.resets + b * a.r_b + r.first * a.r_t;
  if (r.valid == S::STEPS && a.r_t == 1) {
    typedef uint32_t U __attribute__((aligned(1), may_alias));
    const U* q = reinterpret_cast<const U*>(first + lane_rows<S>(j, a.reverse));
#pragma unroll
    for (int k = 0; k < S::L / 4; ++k) p[k] = q[k];
  } else {
#pragma unroll
    for (int k = 0; k < S::L / 4; ++k) p[k] = 0;
#pragma unroll
    for (int i = 0; i < S::L; ++i) {
      const uint32_t v = first[row_offset(j + i, r, a.reverse, (uint32_t)a.r_t, 0)];
      const int at = r.valid == S::STEPS ? step_row<S>(i, a.reverse) : i;
      const uint32_t byte = v && j + i < r.valid ? 1u << (8 * (at & 3)) : 0;
#pragma unroll
      for (int k = 0; k < S::L / 4; ++k) p[k] |= at / 4 == k ? byte : 0;
    }
  }
}
template <int W>
__device__ __forceinline__ bool any_reset(const uint32_t (&p)[W]) {
  uint32_t v = 0;
#pragma unroll
  for (int k = 0; k < W; ++k) v |= p[k];
  return v != 0;
}
// bit i: step i of this lane begins an episode.  In a full tile read backwards the bytes lie backwards.
template <typename S>
__device__ __forceinline__ uint32_t reset_bits(const uint32_t (&p)[S::L / 4], const Rows& r, int reverse) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < S::L; ++i) {
    const int at = r.valid == S::STEPS ? step_row<S>(i, reverse) : i;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < S::L / 4; ++k) w = at / 4 == k ? p[k] : w;
    bits |= ((w >> (8 * (at & 3))) & 0xff ? 1u : 0u) << i;
  }
  return bits;
}

// A lane's channels.  A row's last pack is moved back to end with the row, so every access is a whole
// pack: the channels it shares with its neighbour are computed, and stored, by both alike.  Rows shorter
// than a pack (TINY) are read element by element.
template <int V, bool TINY>
__device__ __forceinline__ int channel_of(int first, int D) {
  return TINY ? first : first < D - V ? first : D - V;
}

// The channels of a workgroup: SLAB of them.  With decays, where the last slab would hold a single one, it takes
// two more from the one before, so that a pack moved back shares its channels with a lane of its own workgroup
// only: one of two workgroups may walk its tiles twice, which rounds differently.
struct Slab {
  int first, width;
};
template <typename S, bool LOGIT>
__device__ __forceinline__ Slab slab_of(int slab, int slabs, int D) {
  const int taken = !LOGIT && slabs > 1 && D % S::SLAB == 1 ? S::V : 0;
  return {slab * S::SLAB - (slab == slabs - 1 ? taken : 0), S::SLAB - (slab == slabs - 2 ? taken : 0)};
}

// the factor and the input of one step; PLAIN: the step is known to lie inside the history
template <typename T, typename G, int V, bool LOGIT, bool PLAIN>
__device__ __forceinline__ void step_of(const Pack<T, V>& px, const Pack<G, V>& pg, bool on, float (&a)[V],
                                        float (&keep)[V], float (&x)[V], float (&in)[V]) {
  unpack<T, V>(px, x);
  unpack<G, V>(pg, a);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if constexpr (LOGIT) {
      gate_of(exp_minus(a[v]), a[v], keep[v]);
      in[v] = keep[v] * x[v];
    } else {
      keep[v] = 1.0f;
      in[v] = x[v];
    }
    if (!PLAIN && !on) {
      a[v] = 1.0f;
      in[v] = 0.0f;
    }
  }
}

// (A, H, R) <- (A, H, R) o (pA, pH, pR); PLAIN: no resets in this wave
template <int V, bool PLAIN>
__device__ __forceinline__ void compose(float (&A)[V], float (&H)[V], bool& R, const float (&pA)[V],
                                        const float (&pH)[V], bool pR) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    H[v] = !PLAIN && R ? H[v] : fmaf(A[v], pH[v], H[v]);
    A[v] = !PLAIN && R ? 0.0f : A[v] * pA[v];
  }
  R = R || pR;
}

// inclusive scan over the groups of a wave, from the first (UP) or the last group on
template <int V, int CL, bool UP, bool PLAIN>
__device__ __forceinline__ void wave_scan(float (&A)[V], float (&H)[V], bool& R, int lane) {
#pragma unroll
  for (int off = CL; off < 64; off *= 2) {
    float pA[V], pH[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      pA[v] = UP ? __shfl_up(A[v], off) : __shfl_down(A[v], off);
      pH[v] = UP ? __shfl_up(H[v], off) : __shfl_down(H[v], off);
    }
    const int pR = PLAIN ? 0 : UP ? __shfl_up((int)R, off) : __shfl_down((int)R, off);
    if (UP ? lane >= off : lane + off < 64) compose<V, PLAIN>(A, H, R, pA, pH, pR != 0);
  }
}

// the state in front of this lane's steps: `in` (in front of the wave), then the groups before it
template <int V, int CL, bool UP, bool PLAIN>
__device__ __forceinline__ void state_in(float (&A)[V], float (&H)[V], bool R, const float* front, int lane,
                                         float (&s)[V]) {
  float in[V];
#pragma unroll
  for (int v = 0; v < V; ++v) in[v] = front[v];
  const int eR = PLAIN ? 0 : UP ? __shfl_up((int)R, CL) : __shfl_down((int)R, CL);
  const bool edge = UP ? lane < CL : lane >= 64 - CL;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float eA = UP ? __shfl_up(A[v], CL) : __shfl_down(A[v], CL);
    const float eH = UP ? __shfl_up(H[v], CL) : __shfl_down(H[v], CL);
    s[v] = edge ? in[v] : !PLAIN && eR ? eH : fmaf(eA, in[v], eH);
  }
}

// The waves' pairs of a tile and the states in front of the waves.
template <int NW, int SLAB>
struct Pairs {
  float A[NW][SLAB], H[NW][SLAB], in[NW][SLAB];
  int R[NW];
};
template <int V, int NW, int SLAB>
__device__ __forceinline__ void put_pair(Pairs<NW, SLAB>& p, int wave, int slot, const float (&A)[V], const float (&H)[V],
                                         bool R) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    p.A[wave][slot + v] = A[v];
    p.H[wave][slot + v] = H[v];
  }
  p.R[wave] = R;
}
// One wave takes the states of the slab, one per lane, through the pairs of all waves; PROD also forms
// the product.
template <int NW, int SLAB, bool UP, bool PROD>
__device__ __forceinline__ void join_waves(Pairs<NW, SLAB>& p, int lane, float& state, float& prod, bool& forgot) {
  if (lane >= SLAB) return;
  constexpr int AHEAD = NW < 4 ? NW : 4;      // pairs read at once: all of them would take 3 NW registers
#pragma unroll 1
  for (int k0 = 0; k0 < NW; k0 += AHEAD) {
    float A[AHEAD], H[AHEAD];
    int R[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int w = UP ? k0 + k : NW - 1 - k0 - k;
      A[k] = p.A[w][lane];
      H[k] = p.H[w][lane];
      R[k] = p.R[w];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      p.in[UP ? k0 + k : NW - 1 - k0 - k][lane] = state;
      const float next = fmaf(A[k], state, H[k]);
      state = R[k] ? H[k] : next;
      if constexpr (PROD) {
        prod = R[k] ? 0.0f : prod * A[k];
        forgot = forgot || R[k];
      }
    }
  }
}

// ---- decays above one --------------------------------------------------------------------------------
// A product of many decays above one passes the range of a float though the states stay inside it: a state of
// zero, or a small one, or decays that shrink again, and infinity times zero is no state.  A workgroup counts how
// far its channels' decays above one could take a product (the sum of their log2), and where that is further
// than MAX_GROWTH it walks its tiles a second time, with products kept as A 2^E, A between 1/2 and 1: every group
// of lanes takes its steps one after another, and one wave takes the groups.  A walk of its own, behind the other
// and in rolled loops: the same arithmetic within the one loop cost histories without such decays 8 to 14 %
// (registers: their loop uses all it may), the look at the decays costs 0 to 3 % (16 x 2048 x 1024 fp32 forwards
// 85.0 -> 87.6 us, bf16 35.5 -> 36.2) and 1 us where a short history is cut.  The second walk takes twice to four
// times the first (1 x 65536 x 512 bf16 forwards 60 us, with decays of 1.01 throughout 206).
constexpr float MAX_GROWTH = 60.0f;      // 2^60: a state of up to 2^67 times such a product is still a float
__device__ __forceinline__ void normalise(float& A, int& E) {
  const int e = E + __builtin_amdgcn_frexp_expf(A);      // zero, infinity and NaN: 0
  A = __builtin_amdgcn_frexp_mantf(A);
  E = e < -(1 << 24) ? -(1 << 24) : e > (1 << 24) ? 1 << 24 : e;
}
__device__ __forceinline__ float apply_wide(float A, int E, float s, float H) {
  return __builtin_ldexpf(A * s, E) + H;
}

// Whether a lane holds a decay above 1 in size.  Of 16-bit ones by their bits, two at once: added to what one lacks
// to the next power of two, everything above one reaches that exponent's top bit, one itself does not.  (A NaN
// may pass unseen; it is a NaN in either walk.)
template <typename G, int V, int L>
__device__ __forceinline__ bool grows(const Pack<G, V> (&g)[L]) {
  if constexpr (sizeof(G) == 4) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < L; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) most = fmaxf(most, fabsf(__uint_as_float(g[i].w[v])));
    return most > 1.0f;
  } else {
    constexpr uint32_t lacks = __is_same(G, bf16_t) ? 0x4000 - 0x3f80 - 1 : 0x4000 - 0x3c00 - 1;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < L; ++i)
#pragma unroll
      for (int k = 0; k < Pack<G, V>::WORDS; ++k) top |= g[i].w[k] + (lacks << 16 | lacks);
    return (top & 0x40004000u) != 0;
  }
}

// Adds up, for each of a lane's channels, how far decays above one could take a product.
template <typename G, int V, int L>
__device__ __forceinline__ void note_growth(float* growth, const Pack<G, V> (&g)[L], int first, int valid) {
  float p[V];
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = 1.0f;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    float f[V];
    unpack<G, V>(g[i], f);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (first + i < valid) p[v] *= fmaxf(fabsf(f[v]), 1.0f);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) growth[v] += __builtin_amdgcn_logf(p[v]);
}
// The pairs of all groups of a tile and the states in front of them.  (`in` holds the growth before a second walk.)
template <int GROUPS, int SLAB>
struct WidePairs {
  float A[GROUPS][SLAB], H[GROUPS][SLAB], in[GROUPS][SLAB];
  int E[GROUPS][SLAB], R[GROUPS];
};
template <int V, int GROUPS, int SLAB>
__device__ __forceinline__ void put_wide(WidePairs<GROUPS, SLAB>& p, int group, int slot, const float (&A)[V], const int (&E)[V],
                                         const float (&H)[V], bool R) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    p.A[group][slot + v] = A[v];
    p.H[group][slot + v] = H[v];
    p.E[group][slot + v] = E[v];
  }
  p.R[group] = R;
}
template <int GROUPS, int SLAB, bool UP, bool PROD>
__device__ __forceinline__ void walk_wide(WidePairs<GROUPS, SLAB>& p, int lane, float& state, float& prod, int& prod_e,
                                          bool& forgot) {
  if (lane >= SLAB) return;
#pragma unroll 1
  for (int k = 0; k < GROUPS; ++k) {
    const int w = UP ? k : GROUPS - 1 - k;
    const float A = p.A[w][lane], H = p.H[w][lane];
    const int E = p.E[w][lane];
    const bool r = p.R[w];
    p.in[w][lane] = state;
    state = r ? H : apply_wide(A, E, state, H);
    if constexpr (PROD) {
      prod = r ? 0.0f : prod * A;
      prod_e = r ? 0 : prod_e + E;
      normalise(prod, prod_e);
      forgot = forgot || r;
    }
  }
}
// behind agg_h, as far as that is behind agg_a
template <typename T, typename G>
__device__ __forceinline__ int32_t* exponents(const RecArgs<T, G>& a) {
  return reinterpret_cast<int32_t*>(a.agg_h + (a.agg_h - a.agg_a));
}
// What the growth of a workgroup's channels asks for.
template <int GROUPS, int SLAB>
__device__ __forceinline__ bool grows_past(const WidePairs<GROUPS, SLAB>& p, int lane, float limit) {
  float sum = 0.0f;
#pragma unroll 1
  for (int k = 0; k < GROUPS; ++k) sum += p.in[k][lane & (SLAB - 1)];
  return __any(!(sum <= limit));
}
// A chunk's pair is kept with its exponent.  Bit 0 of its byte: a reset, which every slab of channels has alike;
// bit 1, a slab's own (so that decays have a byte for each): some exponent is not 0, or the product could be so large
// that as many of them as there are chunks pass MAX_GROWTH.
enum { CHUNK_RESET = 1, CHUNK_WIDE = 2 };
template <typename T, typename G, bool LOGIT>
__device__ __forceinline__ void put_chunk(const RecArgs<T, G>& a, int64_t b, int slab, int chunk, int lane, int own, float A,
                                          int E, float H, bool reset, bool large) {
  const int64_t o = b * a.chunks + chunk;
  a.agg_a[o * a.D + own] = A;
  a.agg_h[o * a.D + own] = H;
  if constexpr (!LOGIT) exponents(a)[o * a.D + own] = E;
  const bool wide = !LOGIT && (large || __any(E != 0));
  if (lane == 0) a.agg_r[LOGIT ? o : o * a.slabs + slab] = (reset ? CHUNK_RESET : 0) | (wide ? CHUNK_WIDE : 0);
}
// What a wave of a decay kernel has met: decays above one among its steps; a wide chunk in front of its own.
enum { GROWS = 1, AFTER_WIDE = 2 };
// A channel's state taken through the chunks in front of this one (UP; behind it, down), one after another.
template <typename T, typename G, bool UP>
__device__ __forceinline__ void walk_chunks(const RecArgs<T, G>& a, int64_t b, int slab, int chunk, int own, float& state) {
  const int first = UP ? 0 : chunk + 1, last = UP ? chunk : a.chunks;
#pragma unroll 1
  for (int k = 0; k < last - first; ++k) {
    const int64_t o = b * a.chunks + (UP ? first + k : last - 1 - k), at = o * a.D + own;
    const float H = a.agg_h[at];
    state = a.agg_r[o * a.slabs + slab] & CHUNK_RESET ? H : apply_wide(a.agg_a[at], exponents(a)[at], state, H);
  }
}
// A lane's place in the slab, as the kernels below compute it, but from an index that the compiler takes for
// another: its values need not live through their loops.
template <typename S, bool TINY>
struct Place {
  int lane, wave, slot, c, own, group;
  bool active, owner;
  __device__ __forceinline__ Place(int slab, int slabs, int D) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    lane = tid & 63;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    slot = (lane & (S::CL - 1)) * S::V;
    const Slab mine = slab_of<S, false>(slab, slabs, D);
    active = slot < mine.width && mine.first + slot < D;
    c = active ? channel_of<S::V, TINY>(mine.first + slot, D) : 0;
    own = channel_of<S::V, TINY>(mine.first + lane / S::V * S::V, D) + lane % S::V;
    owner = wave == 0 && lane < mine.width && mine.first + lane / S::V * S::V < D && own < D;
    group = wave * S::TG + lane / S::CL;
  }
};

// The state in front of a chunk: the composition of the chunks before it (UP; behind it, down), scanned
// like steps, one chunk per group of lanes.
template <typename T, typename G, typename S, bool DECAY, bool UP, bool TINY>
__device__ __forceinline__ void through_chunks(const RecArgs<T, G>& a, Pairs<S::NW, S::SLAB>& pairs, int64_t b, int slab,
                                               int chunk, int lane, int wave, int slot, int c, bool& grown, float& state) {
  constexpr int V = S::V, GROUPS = S::NW * S::TG;
  const int first = UP ? 0 : chunk + 1, last = UP ? chunk : a.chunks;     // [first, last)
  for (int done = 0; done < last - first; done += GROUPS) {
    const int g = wave * S::TG + lane / S::CL;
    const int k = UP ? first + done + g : last - 1 - done - (GROUPS - 1 - g);
    float A[V], H[V], prod = 0.0f;
    bool R = false, forgot = false, wide = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] = 1.0f;
      H[v] = 0.0f;
    }
    if (k >= first && k < last) {
      const int64_t o = b * a.chunks + k;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (!TINY || v < a.D) {
          A[v] = a.agg_a[o * a.D + c + v];
          H[v] = a.agg_h[o * a.D + c + v];
        }
      const int flags = a.agg_r[DECAY ? o * a.slabs + slab : o];
      R = DECAY ? flags & CHUNK_RESET : flags;
      if (DECAY && (flags & CHUNK_WIDE)) wide = true;
    }
    if (DECAY) grown = grown || __any(wide);
    wave_scan<V, S::CL, UP, false>(A, H, R, lane);
    if (UP ? lane >= 64 - S::CL : lane < S::CL) put_pair<V>(pairs, wave, slot, A, H, R);
    __syncthreads();
    if (wave == 0) join_waves<S::NW, S::SLAB, UP, false>(pairs, lane, state, prod, forgot);
    __syncthreads();
  }
}

// Store of one pack: of step j + i of a full tile, whose first row is `first`; and of step s of a history
// of n steps, anywhere.
template <typename S, typename T, bool TINY>
__device__ __forceinline__ void put_row(T* first, int i, int j, int reverse, int c, int D, const Pack<T, S::V>& p) {
  const uint32_t step = (uint32_t)(D * sizeof(T));
  buffer_store<T, S::V, TINY>(buffer_at(first), __umul24(lane_rows<S>(j, reverse), step) + (uint32_t)(c * sizeof(T)),
                              step * step_row<S>(i, reverse), p);
}
template <typename S, typename T, bool TINY>
__device__ __forceinline__ void put_step(T* base, int64_t s, int64_t n, int reverse, int c, int D, const Pack<T, S::V>& p) {
  T* row = base + (reverse && s < n ? n - 1 - s : s) * D + c;
  if constexpr (!TINY) store_pack<T, S::V>(row, p);
  else store_part<T, S::V>(row, p, D);
}

template <bool B>
struct Bool {
  static constexpr bool value = B;
};

// Step k of a tile's rows, loaded by itself: in the rolled loops below few registers are held, as the loops that
// have no decays above one would otherwise spill theirs.
template <typename S, typename T, bool TINY>
__device__ __forceinline__ Pack<T, S::V> load_step(const T* base, int64_t stride, int k, const Rows& r, int reverse, int c) {
  return buffer_load<T, S::V, TINY>(buffer_at(base + r.first * stride),
                                    row_offset(k, r, reverse, (uint32_t)(stride * sizeof(T)), (uint32_t)(c * sizeof(T))), 0);
}
template <typename T, typename G>
__device__ __forceinline__ bool reset_at(const RecArgs<T, G>& a, int64_t b, int k, const Rows& r) {
  return a.resets && k < r.valid && a.resets[b * a.r_b + (r.first + (a.reverse ? r.here - 1 - k : k)) * a.r_t];
}
// one lane's pair
template <int V>
struct WidePair {
  float A[V], H[V];
  int E[V];
  bool R;
  __device__ __forceinline__ WidePair() : R(false) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] = 1.0f;
      H[v] = 0.0f;
      E[v] = 0;
    }
  }
  __device__ __forceinline__ void add(const float (&f)[V], const float (&in)[V], bool r) {
    R = R || r;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      H[v] = r ? in[v] : fmaf(f[v], H[v], in[v]);
      A[v] = r ? 0.0f : A[v] * f[v];
      normalise(A[v], E[v]);
    }
  }
};

// The tiles of a chunk of a history among whose decays some are above one.
template <typename T, typename G, typename S, bool EMIT, bool TINY>
__device__ __forceinline__ void wide_tiles(const RecArgs<T, G>& a, WidePairs<S::NW * S::TG, S::SLAB>& pairs, int64_t b, int64_t n,
                                           int slab, int chunk, int64_t tile0, int64_t tile1, float& state, float& prod,
                                           int& prod_e, bool& forgot) {
  constexpr int V = S::V, L = S::L, GROUPS = S::NW * S::TG;
  const Place<S, TINY> me(slab, a.slabs, a.D);
  const int lane = me.lane, wave = me.wave, slot = me.slot, c = me.c, own = me.own, group = me.group, j = group * L;
  state = EMIT && me.owner && a.h0 ? a.h0[b * a.D + own] : 0.0f;
  prod = 1.0f;
  prod_e = 0;
  forgot = false;
  if (EMIT && me.owner) walk_chunks<T, G, true>(a, b, slab, chunk, own, state);
#pragma unroll 1
  for (int64_t tile = tile0; tile < tile1; ++tile) {
    const Rows rows = rows_of<S>(tile, n, a.reverse);
    float f[V], keep[V], x[V], in[V];
    const auto step = [&](int k) {
      const Pack<T, V> px = load_step<S, T, TINY>(a.x + b * a.x_b, a.x_t, k, rows, a.reverse, c);
      const Pack<G, V> pg = load_step<S, G, TINY>(a.g + b * a.g_b, a.g_t, k, rows, a.reverse, c);
      step_of<T, G, V, false, false>(px, pg, k < rows.valid, f, keep, x, in);
      return reset_at(a, b, k, rows);
    };
    WidePair<V> p;
#pragma unroll 1
    for (int k = j; k < j + L; ++k) {
      const bool r = step(k);
      p.add(f, in, r);
    }
    __syncthreads();        // the pairs of the tile before are done with
    put_wide<V>(pairs, group, slot, p.A, p.E, p.H, p.R);
    __syncthreads();
    if (wave == 0) {
      walk_wide<GROUPS, S::SLAB, true, !EMIT>(pairs, lane, state, prod, prod_e, forgot);
      if (EMIT && a.carries && me.owner) {
        constexpr int PARTS = S::STEPS == Long::STEPS ? KEEP : 1;
#pragma unroll 1
        for (int q = 0; q < PARTS; ++q)
          if (tile * PARTS + q < a.kept)
            a.carries[(b * a.kept + tile * PARTS + q) * a.D + own] = pairs.in[q * (GROUPS / PARTS)][lane];
      }
    }
    if constexpr (EMIT) {
      __syncthreads();
      if (me.active) {
        float s[V];
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = pairs.in[group][slot + v];
#pragma unroll 1
        for (int k = j; k < j + L; ++k) {
          const bool r = step(k);
          float h[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            s[v] = r ? in[v] : fmaf(f[v], s[v], in[v]);
            h[v] = k < rows.valid ? s[v] : 0.0f;
          }
          const int64_t at = tile * S::STEPS + k;
          if (at < a.T_) put_step<S, T, TINY>(a.h + b * a.T_ * a.D, at, n, a.reverse, c, a.D, pack<T, V>(h));
        }
      }
    }
  }
}

// LOGIT gates or decay gates; EMIT: states out, else the pair of a chunk alone
template <typename T, typename G, typename S, bool LOGIT, bool EMIT, bool TINY>
__global__ __launch_bounds__(S::NW * 64) void recurrence_kernel(RecArgs<T, G> a) {
  constexpr int V = S::V, SLAB = S::SLAB, NW = S::NW, CL = S::CL, L = S::L;
  __shared__ Pairs<NW, SLAB> pairs;
  __shared__ WidePairs<LOGIT ? 1 : NW * S::TG, SLAB> wide;
  __shared__ int wave_grown[NW];      // decays: GROWS, AFTER_WIDE
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slab = blockIdx.x % a.slabs, chunk = blockIdx.x / a.slabs;
  const int slot = (lane & (CL - 1)) * V;
  const Slab mine = slab_of<S, LOGIT>(slab, a.slabs, a.D);
  const bool active = slot < mine.width && mine.first + slot < a.D;
  const int c = active ? channel_of<V, TINY>(mine.first + slot, a.D) : 0;
  // lane k of wave 0 carries the state of this channel
  const int own = channel_of<V, TINY>(mine.first + lane / V * V, a.D) + lane % V;
  const bool owner = wave == 0 && lane < mine.width && mine.first + lane / V * V < a.D && own < a.D;
  const int j = (wave * S::TG + lane / CL) * L;             // this lane's first step in a tile
  const int64_t tile0 = chunk * a.chunk_tiles;
  const int64_t tile1 = tile0 + a.chunk_tiles < a.tiles ? tile0 + a.chunk_tiles : a.tiles;
  for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y) {
    int64_t n = a.T_;
    if (a.lengths) {
      const int64_t len = __builtin_amdgcn_readfirstlane(a.lengths[b]);
      n = len < 0 ? 0 : len > n ? n : len;
    }
    const T* xb = a.x + b * a.x_b;
    const G* gb = a.g + b * a.g_b;
    Tile<T, G, S> cur;
    Rows rows = rows_of<S>(tile0, n, a.reverse);
    load_rows<S, T, TINY>(cur.x, xb, a.x_t, j, rows, a.reverse, c);
    load_rows<S, G, TINY>(cur.g, gb, a.g_t, j, rows, a.reverse, c);
    load_resets<S>(cur.resets, a, b, j, rows);
    float state = EMIT && owner && a.h0 ? a.h0[b * a.D + own] : 0.0f, prod = 1.0f;
    bool forgot = false, grown = false;
    if (EMIT && chunk) through_chunks<T, G, S, !LOGIT, true, TINY>(a, pairs, b, slab, chunk, lane, wave, slot, c, grown, state);
    if constexpr (!LOGIT) {
      wave_grown[wave] = grown ? AFTER_WIDE : 0;
#pragma unroll
      for (int v = 0; v < V; ++v) wide.in[j / L][slot + v] = 0.0f;
    }
    for (int64_t tile = tile0; tile < tile1; ++tile) {
      Tile<T, G, S> next;
      const Rows after = rows_of<S>(tile + 1 < tile1 ? tile + 1 : tile, n, a.reverse);
      load_rows<S, T, TINY>(next.x, xb, a.x_t, j, after, a.reverse, c);
      load_resets<S>(next.resets, a, b, j, after);

      // Most waves of most tiles have no reset and no step behind the end; without the selects for
      // those a step costs half the instructions.
      bool above = false;
      if constexpr (!LOGIT) above = grows<G, V, L>(cur.g);
      const bool plain = rows.valid == S::STEPS && !__any(any_reset(cur.resets) || above);
      if constexpr (!LOGIT)
        if (!plain && __any(above)) {
          wave_grown[wave] |= GROWS;
          note_growth<G, V, L>(&wide.in[j / L][slot], cur.g, j, rows.valid);
        }
      uint32_t resets = 0;
      float A[L][V], H[L][V], sA[V], sH[V];
      bool sR = false;
      const auto scan = [&](auto is_plain) {
        constexpr bool PLAIN = decltype(is_plain)::value;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          float f[V], keep[V], x[V], in[V];
          step_of<T, G, V, LOGIT, PLAIN>(cur.x[i], cur.g[i], j + i < rows.valid, f, keep, x, in);
          const bool r = !PLAIN && ((resets >> i) & 1);
          sR = sR || r;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            A[i][v] = r ? 0.0f : i ? f[v] * A[i ? i - 1 : 0][v] : f[v];
            H[i][v] = (r || !i) ? in[v] : fmaf(f[v], H[i ? i - 1 : 0][v], in[v]);
          }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          sA[v] = A[L - 1][v];
          sH[v] = H[L - 1][v];
        }
        wave_scan<V, CL, true, PLAIN>(sA, sH, sR, lane);
      };
      if (plain) {
        scan(Bool<true>());
      } else {
        resets = reset_bits<S>(cur.resets, rows, a.reverse);
        scan(Bool<false>());
      }
      if (lane >= 64 - CL) put_pair<V>(pairs, wave, slot, sA, sH, sR);
      __syncthreads();
      // part of the next tile's loads only here: all at its start would leave the memory idle once they are in
      load_rows<S, G, TINY>(next.g, gb, a.g_t, j, after, a.reverse, c);
      if (wave == 0) {
        join_waves<NW, SLAB, true, !EMIT>(pairs, lane, state, prod, forgot);
        if (EMIT && a.carries && owner) {
          // a state for each of the gradient's tiles, which are shorter: those in front of some waves
          constexpr int PARTS = S::STEPS == Long::STEPS ? KEEP : 1;
#pragma unroll
          for (int q = 0; q < PARTS; ++q)
            if (tile * PARTS + q < a.kept)
              a.carries[(b * a.kept + tile * PARTS + q) * a.D + own] = pairs.in[q * (NW / PARTS)][lane];
        }
      }
      __syncthreads();
      if constexpr (EMIT) {
        const auto emit = [&](auto is_plain) {
          constexpr bool PLAIN = decltype(is_plain)::value;
          float s[V];
          state_in<V, CL, true, PLAIN>(sA, sH, sR, &pairs.in[wave][slot], lane, s);
          if (active) {
            T* const base = a.h + b * a.T_ * a.D;
            bool r = false;
#pragma unroll
            for (int i = 0; i < L; ++i) {
              r = !PLAIN && (r || ((resets >> i) & 1));
              float h[V];
#pragma unroll
              for (int v = 0; v < V; ++v) {
                h[v] = r ? H[i][v] : fmaf(A[i][v], s[v], H[i][v]);
                if (!PLAIN && j + i >= rows.valid) h[v] = 0.0f;
              }
              const Pack<T, V> p = pack<T, V>(h);
              const int64_t step = tile * S::STEPS + j + i;
              if (PLAIN) put_row<S, T, TINY>(base + rows.first * a.D, i, j, a.reverse, c, a.D, p);
              else if (step < a.T_) put_step<S, T, TINY>(base, step, n, a.reverse, c, a.D, p);
            }
          }
        };
        if (plain) emit(Bool<true>());
        else emit(Bool<false>());
      }
      cur = next;
      rows = after;
    }
    int prod_e = 0;
    bool large = false;
    if constexpr (!LOGIT) {
      // the same answers in every wave: each looks at all of them, and at all channels
      const int grew = lane < NW ? wave_grown[lane & (NW - 1)] : 0;
      bool again = __any(grew & AFTER_WIDE);
      if (__any(grew & GROWS)) {
        again = again || grows_past(wide, lane, MAX_GROWTH);
        if (!EMIT) large = grows_past(wide, lane, MAX_GROWTH / a.chunks);
      }
      if (again)
        wide_tiles<T, G, S, EMIT, TINY>(a, wide, b, n, slab, chunk, tile0, tile1, state, prod, prod_e, forgot);
      if (b + gridDim.y < a.B) __syncthreads();                  // before the flags are written again
    }
    if (owner) {
      if constexpr (EMIT) {
        if (a.last && chunk == a.chunks - 1) a.last[b * a.D + own] = state;
      } else {
        put_chunk<T, G, LOGIT>(a, b, slab, chunk, lane, own, prod, prod_e, state, forgot, large);
      }
    }
  }
}

// One step, no scan: a lane per V channels, each channel one lane's alone, which reads its state before it
// writes the new one: `last` may be h0.
template <typename T, typename G, bool LOGIT>
__global__ __launch_bounds__(256) void step_kernel(RecArgs<T, G> a) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t per_row = (a.D + V - 1) / V;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t b = i / per_row;
  const int c = (int)(i - b * per_row) * V;
  if (b >= a.B) return;
  const int left = a.D - c;
  const bool on = !a.lengths || a.lengths[b] > 0;
  const bool r = a.resets && a.resets[b * a.r_b];
  Pack<T, V> px;
  Pack<G, V> pg;
  px = left >= V ? load_pack<T, V>(a.x + b * a.x_b + c) : load_part<T, V>(a.x + b * a.x_b + c, left);
  pg = left >= V ? load_pack<G, V>(a.g + b * a.g_b + c) : load_part<G, V>(a.g + b * a.g_b + c, left);
  float f[V], keep[V], x[V], in[V], h[V], old[V];
  step_of<T, G, V, LOGIT, true>(px, pg, true, f, keep, x, in);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    old[v] = a.h0 && v < left ? a.h0[b * a.D + c + v] : 0.0f;
    h[v] = r ? in[v] : fmaf(f[v], old[v], in[v]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v < left) {
      if (a.carries) a.carries[b * a.D + c + v] = old[v];
      if (a.last) a.last[b * a.D + c + v] = on ? h[v] : old[v];
    }
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = on ? h[v] : 0.0f;
  const Pack<T, V> p = pack<T, V>(h);
  T* dst = a.h + b * a.D + c;
  if (left >= V) store_pack<T, V>(dst, p);
  else store_part<T, V>(dst, p, left);
}

// The same backwards.  `before` holds the state in front of every step of a tile.
template <typename T, typename G, typename S, bool EMIT, bool TINY>
__device__ __forceinline__ void wide_tiles_grad(const RecArgs<T, G>& a, WidePairs<S::NW * S::TG, S::SLAB>& fw,
                                                WidePairs<S::NW * S::TG, S::SLAB>& bw, float (*before)[S::SLAB], int64_t b,
                                                int64_t n, int slab, int chunk, int64_t tile0, int64_t tile1, float& back,
                                                float& prod, int& prod_e, bool& forgot) {
  constexpr int V = S::V, L = S::L, GROUPS = S::NW * S::TG;
  const Place<S, TINY> me(slab, a.slabs, a.D);
  const int lane = me.lane, wave = me.wave, slot = me.slot, c = me.c, own = me.own, group = me.group, j = group * L;
  back = EMIT && me.owner && a.d_last ? a.d_last[b * a.D + own] : 0.0f;
  prod = 1.0f;
  prod_e = 0;
  forgot = false;
  if (EMIT && me.owner) walk_chunks<T, G, false>(a, b, slab, chunk, own, back);
#pragma unroll 1
  for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
    const Rows rows = rows_of<S>(tile, n, a.reverse);
    float carry = EMIT && me.owner ? a.carries[(b * a.tiles + tile) * a.D + own] : 0.0f;     // the state in front of the tile
    float f[V], keep[V], x[V], in[V], d[V];
    const auto step = [&](int k, bool with_x, bool with_d) {
      Pack<T, V> px, pd;
#pragma unroll
      for (int i = 0; i < Pack<T, V>::WORDS; ++i) px.w[i] = pd.w[i] = 0;
      if (with_x) px = load_step<S, T, TINY>(a.x + b * a.x_b, a.x_t, k, rows, a.reverse, c);
      if (with_d && a.dh && k < rows.valid) pd = load_step<S, T, TINY>(a.dh + b * a.dh_b, a.dh_t, k, rows, a.reverse, c);
      const Pack<G, V> pg = load_step<S, G, TINY>(a.g + b * a.g_b, a.g_t, k, rows, a.reverse, c);
      step_of<T, G, V, false, false>(px, pg, k < rows.valid, f, keep, x, in);
      unpack<T, V>(pd, d);
      return reset_at(a, b, k, rows);
    };
    WidePair<V> p;
#pragma unroll 1
    for (int k = j; k < j + L; ++k) {
      const bool r = step(k, EMIT, false);
      p.add(f, in, r);
    }
    float C[V];
#pragma unroll
    for (int v = 0; v < V; ++v) C[v] = 0.0f;
#pragma unroll 1
    for (int k = j + L - 1; k >= j; --k) {
      const bool r = step(k, false, true);
#pragma unroll
      for (int v = 0; v < V; ++v) C[v] = r ? 0.0f : f[v] * (d[v] + C[v]);
    }
    __syncthreads();        // the pairs of the tile before are done with
    put_wide<V>(bw, group, slot, p.A, p.E, C, p.R);
    if (EMIT) put_wide<V>(fw, group, slot, p.A, p.E, p.H, p.R);
    __syncthreads();
    if (wave == 0) {
      walk_wide<GROUPS, S::SLAB, false, !EMIT>(bw, lane, back, prod, prod_e, forgot);
      if (EMIT) walk_wide<GROUPS, S::SLAB, true, false>(fw, lane, carry, prod, prod_e, forgot);
    }
    if constexpr (EMIT) {
      __syncthreads();
      if (me.active) {
        const int64_t base = b * a.T_ * a.D;
        float s[V];
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = fw.in[group][slot + v];
#pragma unroll 1
        for (int k = j; k < j + L; ++k) {
          const bool r = step(k, true, false);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            before[k][slot + v] = r ? 0.0f : s[v];
            s[v] = r ? in[v] : fmaf(f[v], s[v], in[v]);
          }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = bw.in[group][slot + v];
#pragma unroll 1
        for (int k = j + L - 1; k >= j; --k) {
          const bool r = step(k, false, true), on = k < rows.valid;
          float dx[V], dg[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float grad = d[v] + s[v];
            dx[v] = on ? grad : 0.0f;
            dg[v] = on ? grad * before[k][slot + v] : 0.0f;
            s[v] = r ? 0.0f : f[v] * grad;
          }
          const int64_t at = tile * S::STEPS + k;
          if (at < a.T_) {
            put_step<S, T, TINY>(a.dx + base, at, n, a.reverse, c, a.D, pack<T, V>(dx));
            put_step<S, G, TINY>(a.dg + base, at, n, a.reverse, c, a.D, pack<G, V>(dg));
          }
        }
      }
    }
  }
}

// EMIT: gradients out; else the pair of a chunk's adjoint c_{t-1} = a_t (dh_t + c_t) alone.
template <typename T, typename G, typename S, bool LOGIT, bool EMIT, bool TINY>
__global__ __launch_bounds__(S::NW * 64) void recurrence_grad_kernel(RecArgs<T, G> a) {
  constexpr int V = S::V, SLAB = S::SLAB, NW = S::NW, CL = S::CL, L = S::L;
  __shared__ Pairs<NW, SLAB> fw, bw;
  __shared__ WidePairs<LOGIT ? 1 : NW * S::TG, SLAB> wide_fw, wide_bw;
  __shared__ float before_steps[LOGIT || !EMIT ? 1 : S::STEPS][SLAB];
  __shared__ int wave_grown[NW];      // decays: GROWS, AFTER_WIDE
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slab = blockIdx.x % a.slabs;
  const int chunk = blockIdx.x / a.slabs + (EMIT ? 0 : 1);   // the first chunk's pair is not needed
  const int slot = (lane & (CL - 1)) * V;
  const Slab mine = slab_of<S, LOGIT>(slab, a.slabs, a.D);
  const bool active = slot < mine.width && mine.first + slot < a.D;
  const int c = active ? channel_of<V, TINY>(mine.first + slot, a.D) : 0;
  // lane k of wave 0 carries the adjoint of this channel, lane k of the next wave (if there is one) its state
  constexpr int STATE_WAVE = NW > 1 ? 1 : 0;
  const int own = channel_of<V, TINY>(mine.first + lane / V * V, a.D) + lane % V;
  const bool owns = lane < mine.width && mine.first + lane / V * V < a.D && own < a.D;
  const bool owner = owns && wave == 0, stater = owns && wave == STATE_WAVE;
  const int j = (wave * S::TG + lane / CL) * L;
  const int64_t tile0 = chunk * a.chunk_tiles;
  const int64_t tile1 = tile0 + a.chunk_tiles < a.tiles ? tile0 + a.chunk_tiles : a.tiles;
  for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y) {
    int64_t n = a.T_;
    if (a.lengths) {
      const int64_t len = __builtin_amdgcn_readfirstlane(a.lengths[b]);
      n = len < 0 ? 0 : len > n ? n : len;
    }
    const T* xb = a.x + b * a.x_b;
    const G* gb = a.g + b * a.g_b;
    const T* db = a.dh ? a.dh + b * a.dh_b : xb;      // no gradient of h: any rows, then zeros
    const int64_t d_t = a.dh ? a.dh_t : a.x_t;
    Tile<T, G, S> cur;
    Pack<T, V> dcur[L];
    Rows rows = rows_of<S>(tile1 - 1, n, a.reverse);
    if constexpr (EMIT) load_rows<S, T, TINY>(cur.x, xb, a.x_t, j, rows, a.reverse, c);
    load_rows<S, G, TINY>(cur.g, gb, a.g_t, j, rows, a.reverse, c);
    load_rows<S, T, TINY>(dcur, db, d_t, j, rows, a.reverse, c);
    load_resets<S>(cur.resets, a, b, j, rows);
    // the kept state in front of the tile
    float carry = EMIT && stater ? a.carries[(b * a.tiles + tile1 - 1) * a.D + own] : 0.0f;
    float back = EMIT && owner && a.d_last ? a.d_last[b * a.D + own] : 0.0f, prod = 1.0f;
    bool forgot = false, grown = false;
    if (EMIT && chunk + 1 < a.chunks)
      through_chunks<T, G, S, !LOGIT, false, TINY>(a, bw, b, slab, chunk, lane, wave, slot, c, grown, back);
    if constexpr (!LOGIT) {
      wave_grown[wave] = grown ? AFTER_WIDE : 0;
#pragma unroll
      for (int v = 0; v < V; ++v) wide_bw.in[j / L][slot + v] = 0.0f;
    }
    for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
      Tile<T, G, S> next;
      Pack<T, V> dnext[L];
      const int64_t tile_next = tile > tile0 ? tile - 1 : tile;
      const Rows after = rows_of<S>(tile_next, n, a.reverse);
      if constexpr (EMIT) load_rows<S, T, TINY>(next.x, xb, a.x_t, j, after, a.reverse, c);
      load_resets<S>(next.resets, a, b, j, after);
      const float next_carry = EMIT && stater ? a.carries[(b * a.tiles + tile_next) * a.D + own] : 0.0f;
      if (!a.dh) {
#pragma unroll
        for (int i = 0; i < L; ++i)
#pragma unroll
          for (int k = 0; k < Pack<T, V>::WORDS; ++k) dcur[i].w[k] = 0;
      }
      if constexpr (!EMIT) {
#pragma unroll
        for (int i = 0; i < L; ++i)
#pragma unroll
          for (int k = 0; k < Pack<T, V>::WORDS; ++k) cur.x[i].w[k] = 0;
      }

      bool above = false;
      if constexpr (!LOGIT) above = grows<G, V, L>(cur.g);
      const bool plain = rows.valid == S::STEPS && !__any(any_reset(cur.resets) || above);
      if constexpr (!LOGIT)
        if (!plain && __any(above)) {
          wave_grown[wave] |= GROWS;
          note_growth<G, V, L>(&wide_bw.in[j / L][slot], cur.g, j, rows.valid);
        }
      uint32_t resets = 0;
      float A[V], H[V], C[V], bA[V];     // this lane's pairs: forwards (A, H) and the adjoint's (bA, C)
      float e[L][V];                     // exp(-gate), or the decay itself: half the registers of a and 1 - a
      bool fR = false, bR = false;
      // factor, 1 - factor and input of step i
      const auto step = [&](auto is_plain, int i, float (&f)[V], float (&keep)[V], float (&x)[V], float (&in)[V]) {
        constexpr bool PLAIN = decltype(is_plain)::value;
        unpack<T, V>(cur.x[i], x);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if constexpr (LOGIT) {
            gate_of(e[i][v], f[v], keep[v]);
            in[v] = keep[v] * x[v];
          } else {
            f[v] = e[i][v];
            keep[v] = 1.0f;
            in[v] = x[v];
          }
          if (!PLAIN && j + i >= rows.valid) {
            f[v] = 1.0f;
            in[v] = 0.0f;
          }
        }
      };
      const auto scan = [&](auto is_plain) {
        constexpr bool PLAIN = decltype(is_plain)::value;
        bool R = false;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          A[v] = 1.0f;
          H[v] = C[v] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
          float f[V], keep[V], x[V], in[V], d[V];
          unpack<G, V>(cur.g[i], e[i]);
          if constexpr (LOGIT)
#pragma unroll
            for (int v = 0; v < V; ++v) e[i][v] = exp_minus(e[i][v]);
          step(is_plain, i, f, keep, x, in);
          unpack<T, V>(dcur[i], d);
          const bool r = !PLAIN && ((resets >> i) & 1);
          R = R || r;
          // the adjoint in front of these steps: each one's own gradient times the factors up to it
#pragma unroll
          for (int v = 0; v < V; ++v) {
            if (!PLAIN && j + i >= rows.valid) d[v] = 0.0f;
            H[v] = r ? in[v] : fmaf(f[v], H[v], in[v]);
            A[v] = r ? 0.0f : A[v] * f[v];
            C[v] = !PLAIN && R ? C[v] : fmaf(A[v], d[v], C[v]);
          }
        }
        fR = bR = R;
#pragma unroll
        for (int v = 0; v < V; ++v) bA[v] = A[v];
        wave_scan<V, CL, false, PLAIN>(bA, C, bR, lane);
        if constexpr (EMIT) wave_scan<V, CL, true, PLAIN>(A, H, fR, lane);
      };
      if (plain) {
        scan(Bool<true>());
      } else {
        resets = reset_bits<S>(cur.resets, rows, a.reverse);
        scan(Bool<false>());
      }
      if (lane < CL) put_pair<V>(bw, wave, slot, bA, C, bR);
      if (EMIT && lane >= 64 - CL) put_pair<V>(fw, wave, slot, A, H, fR);
      __syncthreads();
      load_rows<S, G, TINY>(next.g, gb, a.g_t, j, after, a.reverse, c);
      if (wave == 0) join_waves<NW, SLAB, false, !EMIT>(bw, lane, back, prod, forgot);
      if (EMIT && wave == STATE_WAVE) join_waves<NW, SLAB, true, false>(fw, lane, carry, prod, forgot);
      __syncthreads();
      load_rows<S, T, TINY>(dnext, db, d_t, j, after, a.reverse, c);
      if constexpr (EMIT) {
        const auto emit = [&](auto is_plain) {
          constexpr bool PLAIN = decltype(is_plain)::value;
          float before[L][V], s[V], bk[V];
          state_in<V, CL, true, PLAIN>(A, H, fR, &fw.in[wave][slot], lane, s);
          state_in<V, CL, false, PLAIN>(bA, C, bR, &bw.in[wave][slot], lane, bk);
          if (active) {
            const int64_t base = b * a.T_ * a.D;
#pragma unroll
            for (int i = 0; i < L; ++i) {
              float f[V], keep[V], x[V], in[V];
              step(is_plain, i, f, keep, x, in);
              const bool r = !PLAIN && ((resets >> i) & 1);
#pragma unroll
              for (int v = 0; v < V; ++v) {
                before[i][v] = r ? 0.0f : s[v];
                s[v] = r ? in[v] : fmaf(f[v], s[v], in[v]);
              }
            }
#pragma unroll
            for (int i = L - 1; i >= 0; --i) {
              float f[V], keep[V], x[V], in[V], d[V], dx[V], dg[V];
              step(is_plain, i, f, keep, x, in);
              unpack<T, V>(dcur[i], d);
              const bool r = !PLAIN && ((resets >> i) & 1);
#pragma unroll
              for (int v = 0; v < V; ++v) {
                if (!PLAIN && j + i >= rows.valid) d[v] = 0.0f;
                const float grad = d[v] + bk[v];
                if constexpr (LOGIT) {
                  dx[v] = keep[v] * grad;
                  dg[v] = f[v] * dx[v] * (before[i][v] - x[v]);
                } else {
                  dx[v] = grad;
                  dg[v] = grad * before[i][v];
                }
                if (!PLAIN && j + i >= rows.valid) dx[v] = dg[v] = 0.0f;
                bk[v] = r ? 0.0f : f[v] * grad;
              }
              const Pack<T, V> px = pack<T, V>(dx);
              const Pack<G, V> pg = pack<G, V>(dg);
              const int64_t s_i = tile * S::STEPS + j + i;
              if (PLAIN) {
                put_row<S, T, TINY>(a.dx + base + rows.first * a.D, i, j, a.reverse, c, a.D, px);
                put_row<S, G, TINY>(a.dg + base + rows.first * a.D, i, j, a.reverse, c, a.D, pg);
              } else if (s_i < a.T_) {
                put_step<S, T, TINY>(a.dx + base, s_i, n, a.reverse, c, a.D, px);
                put_step<S, G, TINY>(a.dg + base, s_i, n, a.reverse, c, a.D, pg);
              }
            }
          }
        };
        if (plain) emit(Bool<true>());
        else emit(Bool<false>());
      }
      cur = next;
      rows = after;
      carry = next_carry;
#pragma unroll
      for (int i = 0; i < L; ++i) dcur[i] = dnext[i];
    }
    int prod_e = 0;
    bool large = false;
    if constexpr (!LOGIT) {
      // the same answers in every wave: each looks at all of them, and at all channels
      const int grew = lane < NW ? wave_grown[lane & (NW - 1)] : 0;
      bool again = __any(grew & AFTER_WIDE);
      if (__any(grew & GROWS)) {
        again = again || grows_past(wide_bw, lane, MAX_GROWTH);
        if (!EMIT) large = grows_past(wide_bw, lane, MAX_GROWTH / a.chunks);
      }
      if (again)
        wide_tiles_grad<T, G, S, EMIT, TINY>(a, wide_fw, wide_bw, before_steps, b, n, slab, chunk, tile0, tile1, back, prod,
                                             prod_e, forgot);
      if (b + gridDim.y < a.B) __syncthreads();                  // before the flags are written again
    }
    if (owner) {
      if constexpr (EMIT) {
        if (a.dh0 && chunk == 0) a.dh0[b * a.D + own] = back;
      } else {
        put_chunk<T, G, LOGIT>(a, b, slab, chunk, lane, own, prod, prod_e, back, forgot, large);
      }
    }
  }
}

struct Split {
  int slabs, chunks;
  int64_t tiles, chunk_tiles;
  int64_t agg_a, agg_h, agg_r, bytes;   // scratch layout
};
// At most half as many workgroups as CUs: the steps are cut, so that there are nearly as many workgroups
// as CUs and no more (one of 16 waves fills a CU's registers, a 257th would wait for a whole chunk).  The pass over the chunks' pairs is another launch and the latency of a
// tile: up to three tiles are walked as they are (7 x 1001 x 257 fp16, four tiles, odd rows: forwards
// 29 us in one piece, 23 us in four).
Split split_of(int64_t B, int64_t T, int D, bool grad) {
  Split s;
  const bool brief = T <= Short::STEPS, middle = T <= Middle::STEPS;
  s.slabs = (int)ceil_div(D, brief ? Short::SLAB : middle ? Middle::SLAB : Long::SLAB);
  s.tiles = ceil_div(T, brief ? Short::STEPS : middle ? Middle::STEPS : grad ? LongGrad::STEPS : Long::STEPS);
  const int64_t groups = B * s.slabs;
  int64_t chunks = groups > 128 || s.tiles <= 3 ? 1 : 256 / groups;
  if (chunks > s.tiles) chunks = s.tiles;
  s.chunk_tiles = ceil_div(s.tiles, chunks);
  s.chunks = (int)ceil_div(s.tiles, s.chunk_tiles);
  const int64_t pairs = s.chunks > 1 ? B * s.chunks * D * 4 : 0;
  s.agg_a = 0;
  s.agg_h = round_up(pairs, 256);
  s.agg_r = 3 * s.agg_h;      // the exponents lie between
  s.bytes = s.chunks > 1 ? s.agg_r + round_up(B * s.chunks * s.slabs, 256) : 0;
  return s;
}

template <typename T, typename G, bool LOGIT, bool TINY>
int run_forward(const RecArgs<T, G>& a, hipStream_t s) {
  if (a.T_ == 1) {
    constexpr int V = 16 / (int)sizeof(T);
    hipLaunchKernelGGL((step_kernel<T, G, LOGIT>), dim3((unsigned)ceil_div(a.B * ceil_div(a.D, V), 256)),
                       dim3(256), 0, s, a);
    PA_LAUNCH_CHECK();
    return PA_OK;
  }
  const unsigned rows = (unsigned)(a.B < 65535 ? a.B : 65535);
  if (a.T_ <= Short::STEPS) {
    hipLaunchKernelGGL((recurrence_kernel<T, G, Short, LOGIT, true, TINY>), dim3(a.slabs, rows),
                       dim3(Short::NW * 64), 0, s, a);
  } else if (a.T_ <= Middle::STEPS) {
    hipLaunchKernelGGL((recurrence_kernel<T, G, Middle, LOGIT, true, TINY>), dim3(a.slabs, rows),
                       dim3(Middle::NW * 64), 0, s, a);
  } else {
    if (a.chunks > 1) {
      hipLaunchKernelGGL((recurrence_kernel<T, G, Long, LOGIT, false, TINY>),
                         dim3(a.slabs * (a.chunks - 1), rows), dim3(Long::NW * 64), 0, s, a);
      PA_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((recurrence_kernel<T, G, Long, LOGIT, true, TINY>), dim3(a.slabs * a.chunks, rows),
                       dim3(Long::NW * 64), 0, s, a);
  }
  PA_LAUNCH_CHECK();
  return PA_OK;
}

template <typename T, typename G, bool LOGIT, bool TINY>
int run_backward(const RecArgs<T, G>& a, hipStream_t s) {
  const unsigned rows = (unsigned)(a.B < 65535 ? a.B : 65535);
  if (a.T_ <= Short::STEPS) {
    hipLaunchKernelGGL((recurrence_grad_kernel<T, G, Short, LOGIT, true, TINY>), dim3(a.slabs, rows),
                       dim3(Short::NW * 64), 0, s, a);
  } else if (a.T_ <= Middle::STEPS) {
    hipLaunchKernelGGL((recurrence_grad_kernel<T, G, Middle, LOGIT, true, TINY>), dim3(a.slabs, rows),
                       dim3(Middle::NW * 64), 0, s, a);
  } else {
    if (a.chunks > 1) {
      hipLaunchKernelGGL((recurrence_grad_kernel<T, G, LongGrad, LOGIT, false, TINY>),
                         dim3(a.slabs * (a.chunks - 1), rows), dim3(LongGrad::NW * 64), 0, s, a);
      PA_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((recurrence_grad_kernel<T, G, LongGrad, LOGIT, true, TINY>), dim3(a.slabs * a.chunks, rows),
                       dim3(LongGrad::NW * 64), 0, s, a);
  }
  PA_LAUNCH_CHECK();
  return PA_OK;
}

template <typename T, typename G, bool LOGIT>
int run_either(const RecArgs<T, G>& a, bool grad, hipStream_t s) {
  if (a.D < Short::V)
    return grad ? run_backward<T, G, LOGIT, true>(a, s) : run_forward<T, G, LOGIT, true>(a, s);
  return grad ? run_backward<T, G, LOGIT, false>(a, s) : run_forward<T, G, LOGIT, false>(a, s);
}

template <typename T, typename G>
int run(const pa_recurrence_args* p, bool grad, hipStream_t s) {
  const Split sp = split_of(p->B, p->T, p->D, grad);
  uint8_t* scratch = reinterpret_cast<uint8_t*>(p->scratch);
  RecArgs<T, G> a;
  a.x = reinterpret_cast<const T*>(p->x); a.x_b = p->x_b; a.x_t = p->x_t;
  a.g = reinterpret_cast<const G*>(p->gate); a.g_b = p->gate_b; a.g_t = p->gate_t;
  a.h0 = p->h0; a.resets = p->resets; a.r_b = p->resets_b; a.r_t = p->resets_t;
  a.lengths = p->lengths; a.B = p->B; a.T_ = p->T; a.D = p->D; a.reverse = p->reverse;
  a.slabs = sp.slabs; a.chunks = sp.chunks; a.chunk_tiles = sp.chunk_tiles; a.tiles = sp.tiles; a.kept = split_of(p->B, p->T, p->D, true).tiles;
  a.agg_a = reinterpret_cast<float*>(scratch + sp.agg_a);
  a.agg_h = reinterpret_cast<float*>(scratch + sp.agg_h);
  a.agg_r = scratch + sp.agg_r;
  a.h = reinterpret_cast<T*>(p->h); a.last = p->last; a.carries = p->carries;
  a.dh = reinterpret_cast<const T*>(p->d_h); a.dh_b = p->d_h_b; a.dh_t = p->d_h_t;
  a.d_last = p->d_last;
  a.dx = reinterpret_cast<T*>(p->d_x); a.dg = reinterpret_cast<G*>(p->d_gate); a.dh0 = p->d_h0;
  return p->gate_logits ? run_either<T, G, true>(a, grad, s) : run_either<T, G, false>(a, grad, s);
}

int dispatch(const pa_recurrence_args* p, bool grad, hipStream_t s) {
  if (p->dtype == PA_F32) return run<float, float>(p, grad, s);
  if (p->dtype == PA_BF16)
    return p->gate_dtype == PA_F32 ? run<bf16_t, float>(p, grad, s) : run<bf16_t, bf16_t>(p, grad, s);
  return p->gate_dtype == PA_F32 ? run<f16_t, float>(p, grad, s) : run<f16_t, f16_t>(p, grad, s);
}

int check_args(const char* who, const pa_recurrence_args* p, bool grad) {
  PA_REQUIRE(p, PA_ERR_INVALID, "%s: null argument", who);
  PA_REQUIRE(elem_size(p->dtype), PA_ERR_UNSUPPORTED, "%s: input dtype %d", who, p->dtype);
  PA_REQUIRE(p->gate_dtype == p->dtype || p->gate_dtype == PA_F32, PA_ERR_UNSUPPORTED,
             "%s: gate dtype %d with input dtype %d (the input's own, or float32)", who, p->gate_dtype, p->dtype);
  const int64_t size = elem_size(p->dtype), gate_size = elem_size(p->gate_dtype), wide = 1 << 23;
  const auto fits = [&](int64_t stride, int64_t bytes) { return stride >= 0 && stride * bytes < wide; };
  PA_REQUIRE(fits(p->D, 4) && fits(p->x_t, size) && fits(p->gate_t, gate_size) && fits(p->resets_t, 1) &&
                 fits(p->d_h_t, size), PA_ERR_UNSUPPORTED, "%s: a step is 2^23 bytes or more from the next", who);
  PA_REQUIRE(p->B >= 0 && p->T >= 1 && p->D >= 1 && p->B <= (1ll << 31) / p->D, PA_ERR_INVALID,
             "%s: bad shape (batch %lld, time %lld, channels %d)", who, (long long)p->B, (long long)p->T, p->D);
  PA_REQUIRE(p->B == 0 || (p->x && p->gate), PA_ERR_INVALID, "%s: null pointer", who);
  PA_REQUIRE(p->B == 0 || p->scratch || split_of(p->B, p->T, p->D, grad).bytes == 0, PA_ERR_INVALID,
             "%s: this shape needs scratch (pa_gated_recurrence_scratch)", who);
  return PA_OK;
}

// Whether `last` lies apart from what the pass reads.  A single step reads a channel before it writes it, so
// there `last` may be h0, or x or the gate in the same layout; anything else would be read by some lanes after
// others have written it.
bool last_is_apart(const pa_recurrence_args* p) {
  if (!p->last) return true;
  const uintptr_t out = reinterpret_cast<uintptr_t>(p->last), out_end = out + p->B * p->D * 4;
  const auto clear_of = [&](const void* in, int64_t last_element, int64_t size) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(in);
    return !in || at >= out_end || at + (last_element + 1) * size <= out;
  };
  const auto rows_clear = [&](const void* in, int64_t b, int64_t t, int64_t size) {
    const bool same = p->T == 1 && in == p->last && size == 4 && (b == p->D || p->B == 1);
    return same || clear_of(in, (p->B - 1) * b + (p->T - 1) * t + p->D - 1, size);
  };
  return rows_clear(p->h0, p->D, 0, 4) && rows_clear(p->x, p->x_b, p->x_t, elem_size(p->dtype)) &&
         rows_clear(p->gate, p->gate_b, p->gate_t, elem_size(p->gate_dtype)) &&
         clear_of(p->resets, (p->B - 1) * p->resets_b + (p->T - 1) * p->resets_t, 1) &&
         clear_of(p->lengths, p->B - 1, 4);
}

}  // namespace

extern "C" int64_t pa_gated_recurrence_scratch(int64_t B, int64_t T, int32_t D) {
  if (B <= 0 || T <= 0 || D <= 0) return 0;
  const int64_t forward = split_of(B, T, D, false).bytes, grad = split_of(B, T, D, true).bytes;
  return forward > grad ? forward : grad;
}

extern "C" int64_t pa_gated_recurrence_carries(int64_t B, int64_t T, int32_t D) {
  return B <= 0 || T <= 0 || D <= 0 ? 0 : B * split_of(B, T, D, true).tiles * D;
}

extern "C" int pa_gated_recurrence(const pa_recurrence_args* args, void* stream) {
  const int rc = check_args("pa_gated_recurrence", args, false);
  if (rc != PA_OK) return rc;
  if (args->B == 0) return PA_OK;
  PA_REQUIRE(args->h, PA_ERR_INVALID, "pa_gated_recurrence: null output");
  PA_REQUIRE(last_is_apart(args), PA_ERR_INVALID, "pa_gated_recurrence: the new state overlaps an input that is still read");
  PA_ON_DEVICE(args->device);
  return dispatch(args, false, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int pa_gated_recurrence_grad(const pa_recurrence_args* args, void* stream) {
  const int rc = check_args("pa_gated_recurrence_grad", args, true);
  if (rc != PA_OK) return rc;
  if (args->B == 0) return PA_OK;
  PA_REQUIRE(args->carries && args->d_x && args->d_gate, PA_ERR_INVALID,
             "pa_gated_recurrence_grad: null pointer (carries, d_x, d_gate)");
  PA_ON_DEVICE(args->device);
  return dispatch(args, true, reinterpret_cast<hipStream_t>(stream));
}
