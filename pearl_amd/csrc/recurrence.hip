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
// A workgroup owns a slab of channels that is one 128-byte line wide in the input's type and walks the
// steps in tiles: 8 lanes side by side in a row of x, 8 groups of L consecutive steps per wave, waves
// behind one another in time.  Each lane scans its own L steps, groups are joined by lane shuffles,
// waves through LDS, the state behind the tile stays in LDS for the next one while that tile's loads
// are already under way.  Every input is read once and every output written once.  The state is fp32
// throughout; only the stored h is rounded to the input's type.
//
// Where batch x channels give too few workgroups, the steps are cut into chunks: a first launch
// composes each chunk's pair, the second starts every chunk from the composition of those before it.
//
// Backward, with G_t = dh_t + c_t and c_{t-1} = a_t G_t (0 at a reset), c_T = d_last:
//   decay:  dx = G, dg = G h_{t-1};   logit:  dx = (1 - a) G, dg = a (1 - a) G (h_{t-1} - x);
//   d_h0 = c_0.  The forward pass keeps the fp32 state in front of every tile (1 / 256 of the steps);
// the states inside a tile are computed again from it rather than read back rounded.
#include "seq_common.hpp"

using namespace pa;
using namespace pa::seq;

namespace {

constexpr int CL = 8;        // lanes side by side in a row
constexpr int TG = 64 / CL;  // groups of consecutive steps per wave

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
  float* agg_a; float* agg_h; uint8_t* agg_r;    // [B][chunks][D], [B][chunks]: the chunks' pairs
  T* h; float* last; float* carries;             // [B][T][D], [B][D] or null, [B][tiles][D] or null
  const T* dh; int64_t dh_b, dh_t;               // or null: zeros
  const float* d_last;                           // [B][D] or null
  T* dx; G* dg; float* dh0;                      // dh0 or null
};

// a and 1 - a of a logit; both to a few ulp, also where one of them is tiny
__device__ __forceinline__ void gate_of(float z, float& a, float& keep) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504088896340736f * fabsf(z));
  const float hi = __builtin_amdgcn_rcpf(1.0f + e), lo = e * hi;
  a = z >= 0.0f ? hi : lo;
  keep = z >= 0.0f ? lo : hi;
  if (z != z) a = keep = z;
}

template <typename T, typename G, int NW, int L>
struct Tile {
  static constexpr int V = 16 / (int)sizeof(T);   // channels per lane
  static constexpr int STEPS = NW * TG * L;
  static constexpr int SLAB = CL * V;
  Pack<T, V> x[L];
  Pack<G, V> g[L];
  uint32_t resets;   // bit i: step i of this lane begins an episode
};

// the place of step `s` of a history of n steps
__device__ __forceinline__ int64_t place_of(int64_t s, int64_t n, int reverse) {
  return reverse && s < n ? n - 1 - s : s;
}

template <typename T, int V, int L>
__device__ __forceinline__ void load_rows(Pack<T, V> (&r)[L], const T* base, int64_t stride, int64_t s0,
                                          int64_t n, int reverse, int left) {
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int64_t s = s0 + i;
#pragma unroll
    for (int k = 0; k < Pack<T, V>::WORDS; ++k) r[i].w[k] = 0;
    if (s < n && left > 0) {
      const T* p = base + place_of(s, n, reverse) * stride;
      r[i] = left >= V ? load_pack<T, V>(p) : load_part<T, V>(p, left);
    }
  }
}

template <typename T, typename G, int L>
__device__ __forceinline__ uint32_t load_resets(const RecArgs<T, G>& a, int64_t b, int64_t s0, int64_t n) {
  uint32_t bits = 0;
  if (a.resets) {
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (s0 + i < n && a.resets[b * a.r_b + place_of(s0 + i, n, a.reverse) * a.r_t]) bits |= 1u << i;
  }
  return bits;
}

// the pair of one step: a = 1, b = 0 where the history has ended
template <typename T, typename G, int V, bool LOGIT>
__device__ __forceinline__ void step_of(const Pack<T, V>& px, const Pack<G, V>& pg, bool on, float (&a)[V],
                                        float (&keep)[V], float (&x)[V]) {
  unpack<T, V>(px, x);
  unpack<G, V>(pg, a);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if constexpr (LOGIT) {
      gate_of(a[v], a[v], keep[v]);
    } else {
      keep[v] = 1.0f;
    }
    if (!on) {
      a[v] = 1.0f;
      keep[v] = 0.0f;
    }
  }
}

// (A, H, R) <- (A, H, R) o (pA, pH, pR)
template <int V>
__device__ __forceinline__ void compose(float (&A)[V], float (&H)[V], bool& R, const float (&pA)[V],
                                        const float (&pH)[V], bool pR) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    H[v] = R ? H[v] : fmaf(A[v], pH[v], H[v]);
    A[v] = R ? 0.0f : A[v] * pA[v];
  }
  R = R || pR;
}

// inclusive scan over the 8 groups of a wave, from the first (UP) or the last group on
template <int V, bool UP>
__device__ __forceinline__ void wave_scan(float (&A)[V], float (&H)[V], bool& R, int lane) {
#pragma unroll
  for (int off = CL; off < 64; off *= 2) {
    float pA[V], pH[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      pA[v] = UP ? __shfl_up(A[v], off) : __shfl_down(A[v], off);
      pH[v] = UP ? __shfl_up(H[v], off) : __shfl_down(H[v], off);
    }
    const int pR = UP ? __shfl_up((int)R, off) : __shfl_down((int)R, off);
    if (UP ? lane >= off : lane + off < 64) compose<V>(A, H, R, pA, pH, pR != 0);
  }
}

// the state in front of this lane's steps: `in` (in front of the wave), then the groups before it
template <int V, bool UP>
__device__ __forceinline__ void state_in(float (&A)[V], float (&H)[V], bool R, const float* in, int lane,
                                         float (&s)[V]) {
  const int eR = UP ? __shfl_up((int)R, CL) : __shfl_down((int)R, CL);
  const bool edge = UP ? lane < CL : lane >= 64 - CL;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float eA = UP ? __shfl_up(A[v], CL) : __shfl_down(A[v], CL);
    const float eH = UP ? __shfl_up(H[v], CL) : __shfl_down(H[v], CL);
    s[v] = edge ? in[v] : eR ? eH : fmaf(eA, in[v], eH);
  }
}

template <typename T, typename G, int NW, int L>
struct Shared {
  static constexpr int SLAB = Tile<T, G, NW, L>::SLAB;
  float A[NW][SLAB], H[NW][SLAB], in[NW][SLAB];
  int R[NW];
};

// LOGIT gates or decay gates; EMIT: states out, else the pair of a chunk alone
template <typename T, typename G, int NW, int L, bool LOGIT, bool EMIT>
__global__ __launch_bounds__(NW * 64) void recurrence_kernel(RecArgs<T, G> a) {
  using Ti = Tile<T, G, NW, L>;
  constexpr int V = Ti::V, SLAB = Ti::SLAB;
  __shared__ Shared<T, G, NW, L> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slab = blockIdx.x % a.slabs, chunk = blockIdx.x / a.slabs;
  const int cl = (lane & (CL - 1)) * V;
  const int c = slab * SLAB + cl;
  const int left = a.D - c;
  const int own = slab * SLAB + tid;                 // the channel whose state thread tid < SLAB carries
  const bool owner = tid < SLAB && own < a.D;
  const int64_t tile0 = chunk * a.chunk_tiles;
  const int64_t tile1 = tile0 + a.chunk_tiles < a.tiles ? tile0 + a.chunk_tiles : a.tiles;
  for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y) {
    int64_t n = a.T_;
    if (a.lengths) {
      n = a.lengths[b];
      n = n < 0 ? 0 : n > a.T_ ? a.T_ : n;
    }
    const T* xb = a.x + b * a.x_b + c;
    const G* gb = a.g + b * a.g_b + c;
    float state = 0.0f, prod = 1.0f;
    bool forgot = false;
    if (EMIT && owner) {
      state = a.h0 ? a.h0[b * a.D + own] : 0.0f;
      for (int k = 0; k < chunk; ++k) {
        const int64_t o = b * a.chunks + k;
        state = a.agg_r[o] ? a.agg_h[o * a.D + own] : fmaf(a.agg_a[o * a.D + own], state, a.agg_h[o * a.D + own]);
      }
    }
    Ti cur;
    int64_t s0 = tile0 * Ti::STEPS + (wave * TG + lane / CL) * L;
    load_rows<T, V, L>(cur.x, xb, a.x_t, s0, n, a.reverse, left);
    load_rows<G, V, L>(cur.g, gb, a.g_t, s0, n, a.reverse, left);
    cur.resets = load_resets<T, G, L>(a, b, s0, n);
    for (int64_t tile = tile0; tile < tile1; ++tile, s0 += Ti::STEPS) {
      Ti next;
      const int64_t s1 = s0 + Ti::STEPS;
      const int64_t lim = tile + 1 < tile1 ? n : 0;   // nothing behind the last tile
      load_rows<T, V, L>(next.x, xb, a.x_t, s1, lim ? n : 0, a.reverse, left);
      load_rows<G, V, L>(next.g, gb, a.g_t, s1, lim ? n : 0, a.reverse, left);
      next.resets = lim ? load_resets<T, G, L>(a, b, s1, n) : 0;

      float A[L][V], H[L][V];
      bool R = false;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        float f[V], keep[V], x[V];
        step_of<T, G, V, LOGIT>(cur.x[i], cur.g[i], s0 + i < n, f, keep, x);
        const bool r = (cur.resets >> i) & 1;
        R = R || r;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float in = s0 + i < n ? (LOGIT ? keep[v] * x[v] : x[v]) : 0.0f;
          A[i][v] = r ? 0.0f : i ? f[v] * A[i ? i - 1 : 0][v] : f[v];
          H[i][v] = (r || !i) ? in : fmaf(f[v], H[i ? i - 1 : 0][v], in);
        }
      }
      float sA[V], sH[V];
      bool sR = R;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        sA[v] = A[L - 1][v];
        sH[v] = H[L - 1][v];
      }
      wave_scan<V, true>(sA, sH, sR, lane);
      if (lane >= 64 - CL) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          sh.A[wave][cl + v] = sA[v];
          sh.H[wave][cl + v] = sH[v];
        }
        if (lane == 63) sh.R[wave] = sR;
      }
      __syncthreads();
      if (tid < SLAB) {
        if (EMIT && a.carries && owner) a.carries[(b * a.tiles + tile) * a.D + own] = state;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          if (EMIT) sh.in[w][tid] = state;
          const bool r = sh.R[w];
          state = r ? sh.H[w][tid] : fmaf(sh.A[w][tid], state, sh.H[w][tid]);
          prod = r ? 0.0f : prod * sh.A[w][tid];
          forgot = forgot || r;
        }
      }
      __syncthreads();
      if constexpr (EMIT) {
        float in[V];
        state_in<V, true>(sA, sH, sR, &sh.in[wave][cl], lane, in);
        bool r = false;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          r = r || ((cur.resets >> i) & 1);
          float h[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            h[v] = r ? H[i][v] : fmaf(A[i][v], in[v], H[i][v]);
            if (s0 + i >= n) h[v] = 0.0f;
          }
          if (s0 + i < a.T_ && left > 0) {
            const Pack<T, V> p = pack<T, V>(h);
            T* dst = a.h + (b * a.T_ + place_of(s0 + i, n, a.reverse)) * a.D + c;
            if (left >= V) store_pack<T, V>(dst, p);
            else store_part<T, V>(dst, p, left);
          }
        }
      }
      cur = next;
    }
    if (owner) {
      if constexpr (EMIT) {
        if (a.last && chunk == a.chunks - 1) a.last[b * a.D + own] = state;
      } else {
        const int64_t o = b * a.chunks + chunk;
        a.agg_a[o * a.D + own] = prod;
        a.agg_h[o * a.D + own] = state;
        if (tid == 0) a.agg_r[o] = forgot;     // the same in every slab
      }
    }
  }
}

// One step, no scan: a lane per V channels.
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
  float f[V], keep[V], x[V], h[V], old[V];
  step_of<T, G, V, LOGIT>(px, pg, true, f, keep, x);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    old[v] = a.h0 && v < left ? a.h0[b * a.D + c + v] : 0.0f;
    const float in = LOGIT ? keep[v] * x[v] : x[v];
    h[v] = r ? in : fmaf(f[v], old[v], in);
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (a.last && v < left) a.last[b * a.D + c + v] = on ? h[v] : old[v];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = on ? h[v] : 0.0f;
  const Pack<T, V> p = pack<T, V>(h);
  T* dst = a.h + b * a.D + c;
  if (left >= V) store_pack<T, V>(dst, p);
  else store_part<T, V>(dst, p, left);
}

// EMIT: gradients out; else the pair of a chunk's adjoint c_{t-1} = a_t (dh_t + c_t) alone.
template <typename T, typename G, int NW, int L, bool LOGIT, bool EMIT>
__global__ __launch_bounds__(NW * 64) void recurrence_grad_kernel(RecArgs<T, G> a) {
  using Ti = Tile<T, G, NW, L>;
  constexpr int V = Ti::V, SLAB = Ti::SLAB;
  __shared__ Shared<T, G, NW, L> fw, bw;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slab = blockIdx.x % a.slabs;
  const int chunk = blockIdx.x / a.slabs + (EMIT ? 0 : 1);   // the first chunk's pair is not needed
  const int cl = (lane & (CL - 1)) * V;
  const int c = slab * SLAB + cl;
  const int left = a.D - c;
  // threads 0 .. SLAB-1 carry the adjoint of a channel; with more than one wave the next ones its state
  const bool two = NW > 1;
  const int own = slab * SLAB + (tid & (SLAB - 1));
  const bool adjoint = tid < SLAB;
  const bool stater = two ? tid >= 64 && tid < 64 + SLAB : tid < SLAB;
  const int64_t tile0 = chunk * a.chunk_tiles;
  const int64_t tile1 = tile0 + a.chunk_tiles < a.tiles ? tile0 + a.chunk_tiles : a.tiles;
  for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y) {
    int64_t n = a.T_;
    if (a.lengths) {
      n = a.lengths[b];
      n = n < 0 ? 0 : n > a.T_ ? a.T_ : n;
    }
    const T* xb = a.x + b * a.x_b + c;
    const G* gb = a.g + b * a.g_b + c;
    const T* db = a.dh ? a.dh + b * a.dh_b + c : nullptr;
    float back = 0.0f, prod = 1.0f;
    bool forgot = false;
    if (EMIT && adjoint && own < a.D) {
      back = a.d_last ? a.d_last[b * a.D + own] : 0.0f;
      for (int k = a.chunks - 1; k > chunk; --k) {
        const int64_t o = b * a.chunks + k;
        back = a.agg_r[o] ? a.agg_h[o * a.D + own] : fmaf(a.agg_a[o * a.D + own], back, a.agg_h[o * a.D + own]);
      }
    }
    Ti cur;
    Pack<T, V> dcur[L];
    int64_t s0 = (tile1 - 1) * Ti::STEPS + (wave * TG + lane / CL) * L;
    if constexpr (EMIT) load_rows<T, V, L>(cur.x, xb, a.x_t, s0, n, a.reverse, left);
    load_rows<G, V, L>(cur.g, gb, a.g_t, s0, n, a.reverse, left);
    load_rows<T, V, L>(dcur, db, a.dh_t, s0, db ? n : 0, a.reverse, left);
    cur.resets = load_resets<T, G, L>(a, b, s0, n);
    for (int64_t tile = tile1 - 1; tile >= tile0; --tile, s0 -= Ti::STEPS) {
      Ti next;
      Pack<T, V> dnext[L];
      const int64_t s1 = s0 - Ti::STEPS;
      const bool more = tile > tile0;
      if constexpr (EMIT) load_rows<T, V, L>(next.x, xb, a.x_t, s1, more ? n : s1, a.reverse, left);
      load_rows<G, V, L>(next.g, gb, a.g_t, s1, more ? n : s1, a.reverse, left);
      load_rows<T, V, L>(dnext, db, a.dh_t, s1, more && db ? n : s1, a.reverse, left);
      next.resets = more ? load_resets<T, G, L>(a, b, s1, n) : 0;
      float state = 0.0f;
      if (EMIT && stater && own < a.D) state = a.carries[(b * a.tiles + tile) * a.D + own];

      // this lane's pairs: forwards (A, H) and the adjoint's (A, C)
      float A[V], H[V], C[V];
      bool R = false;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        A[v] = 1.0f;
        H[v] = C[v] = 0.0f;
      }
      float f[L][V], keep[L][V];
#pragma unroll
      for (int i = 0; i < L; ++i) {
        float x[V];
        if constexpr (!EMIT) {
#pragma unroll
          for (int k = 0; k < Pack<T, V>::WORDS; ++k) cur.x[i].w[k] = 0;
        }
        const bool on = s0 + i < n;
        step_of<T, G, V, LOGIT>(cur.x[i], cur.g[i], on, f[i], keep[i], x);
        const bool r = (cur.resets >> i) & 1;
        R = R || r;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float in = on ? (LOGIT ? keep[i][v] * x[v] : x[v]) : 0.0f;
          H[v] = r ? in : fmaf(f[i][v], H[v], in);
          A[v] = r ? 0.0f : A[v] * f[i][v];
        }
      }
#pragma unroll
      for (int i = L - 1; i >= 0; --i) {
        float d[V];
        unpack<T, V>(dcur[i], d);
        const bool r = (cur.resets >> i) & 1;
#pragma unroll
        for (int v = 0; v < V; ++v) C[v] = r ? 0.0f : f[i][v] * (d[v] + C[v]);
      }
      float bA[V];
      bool fR = R, bR = R;
#pragma unroll
      for (int v = 0; v < V; ++v) bA[v] = A[v];
      wave_scan<V, false>(bA, C, bR, lane);
      if (lane < CL) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          bw.A[wave][cl + v] = bA[v];
          bw.H[wave][cl + v] = C[v];
        }
        if (lane == 0) bw.R[wave] = bR;
      }
      if constexpr (EMIT) {
        wave_scan<V, true>(A, H, fR, lane);
        if (lane >= 64 - CL) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            fw.A[wave][cl + v] = A[v];
            fw.H[wave][cl + v] = H[v];
          }
          if (lane == 63) fw.R[wave] = fR;
        }
      }
      __syncthreads();
      if (adjoint) {
#pragma unroll
        for (int w = NW - 1; w >= 0; --w) {
          if (EMIT) bw.in[w][tid] = back;
          const bool r = bw.R[w];
          back = r ? bw.H[w][tid] : fmaf(bw.A[w][tid], back, bw.H[w][tid]);
          prod = r ? 0.0f : prod * bw.A[w][tid];
          forgot = forgot || r;
        }
      }
      if (EMIT && stater) {
        const int ch = tid & (SLAB - 1);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          fw.in[w][ch] = state;
          state = fw.R[w] ? fw.H[w][ch] : fmaf(fw.A[w][ch], state, fw.H[w][ch]);
        }
      }
      __syncthreads();
      if constexpr (EMIT) {
        float before[L][V], s[V], bk[V];
        state_in<V, true>(A, H, fR, &fw.in[wave][cl], lane, s);
        state_in<V, false>(bA, C, bR, &bw.in[wave][cl], lane, bk);
#pragma unroll
        for (int i = 0; i < L; ++i) {
          float x[V];
          unpack<T, V>(cur.x[i], x);
          const bool r = (cur.resets >> i) & 1;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            before[i][v] = r ? 0.0f : s[v];
            const float in = s0 + i < n ? (LOGIT ? keep[i][v] * x[v] : x[v]) : 0.0f;
            s[v] = r ? in : fmaf(f[i][v], s[v], in);
          }
        }
#pragma unroll
        for (int i = L - 1; i >= 0; --i) {
          float x[V], d[V], dx[V], dg[V];
          unpack<T, V>(cur.x[i], x);
          unpack<T, V>(dcur[i], d);
          const bool r = (cur.resets >> i) & 1;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float grad = d[v] + bk[v];
            if constexpr (LOGIT) {
              dx[v] = keep[i][v] * grad;
              dg[v] = f[i][v] * dx[v] * (before[i][v] - x[v]);
            } else {
              dx[v] = grad;
              dg[v] = grad * before[i][v];
            }
            if (s0 + i >= n) dx[v] = dg[v] = 0.0f;
            bk[v] = r ? 0.0f : f[i][v] * grad;
          }
          if (s0 + i < a.T_ && left > 0) {
            const int64_t o = (b * a.T_ + place_of(s0 + i, n, a.reverse)) * a.D + c;
            const Pack<T, V> px = pack<T, V>(dx);
            const Pack<G, V> pg = pack<G, V>(dg);
            if (left >= V) {
              store_pack<T, V>(a.dx + o, px);
              store_pack<G, V>(a.dg + o, pg);
            } else {
              store_part<T, V>(a.dx + o, px, left);
              store_part<G, V>(a.dg + o, pg, left);
            }
          }
        }
      }
      cur = next;
#pragma unroll
      for (int i = 0; i < L; ++i) dcur[i] = dnext[i];
    }
    if (adjoint && own < a.D) {
      if constexpr (EMIT) {
        if (a.dh0 && chunk == 0) a.dh0[b * a.D + own] = back;
      } else {
        const int64_t o = b * a.chunks + chunk;
        a.agg_a[o * a.D + own] = prod;
        a.agg_h[o * a.D + own] = back;
        if (tid == 0) a.agg_r[o] = forgot;
      }
    }
  }
}

// Steps per tile: the forward and the backward pass agree on it, the kept states lie between tiles.
// Histories of up to 32 steps take one wave per slab, longer ones eight.
constexpr int SHORT = TG * 4;
int64_t tile_steps(int64_t T) { return T <= SHORT ? SHORT : 8 * TG * 4; }

struct Split {
  int slabs, chunks;
  int64_t tiles, chunk_tiles;
  int64_t agg_a, agg_h, agg_r, bytes;   // scratch layout
};
Split split_of(int64_t B, int64_t T, int D, int dtype) {
  Split s;
  const int slab = CL * 16 / elem_size(dtype);
  s.slabs = (int)ceil_div(D, slab);
  s.tiles = ceil_div(T, tile_steps(T));
  const int64_t groups = B * s.slabs;
  int64_t chunks = groups >= 192 ? 1 : ceil_div(512, groups);
  if (chunks > s.tiles) chunks = s.tiles;
  if (chunks > 128) chunks = 128;
  if (chunks < 1) chunks = 1;
  s.chunk_tiles = ceil_div(s.tiles, chunks);
  s.chunks = (int)ceil_div(s.tiles, s.chunk_tiles);
  if (s.chunks < 1) s.chunks = 1;
  const int64_t pairs = s.chunks > 1 ? B * s.chunks * D * 4 : 0;
  s.agg_a = 0;
  s.agg_h = round_up(pairs, 256);
  s.agg_r = 2 * s.agg_h;
  s.bytes = s.chunks > 1 ? s.agg_r + round_up(B * s.chunks, 256) : 0;
  return s;
}

template <typename T, typename G, bool LOGIT>
int run_forward(const pa_recurrence_args* p, const RecArgs<T, G>& a, hipStream_t s) {
  if (a.T_ == 1 && !a.carries) {
    constexpr int V = 16 / (int)sizeof(T);
    hipLaunchKernelGGL((step_kernel<T, G, LOGIT>), dim3((unsigned)ceil_div(a.B * ceil_div(a.D, V), 256)),
                       dim3(256), 0, s, a);
    PA_LAUNCH_CHECK();
    return PA_OK;
  }
  const unsigned rows = (unsigned)(a.B < 65535 ? a.B : 65535);
  if (a.T_ <= SHORT) {
    hipLaunchKernelGGL((recurrence_kernel<T, G, 1, 4, LOGIT, true>), dim3(a.slabs, rows), dim3(64), 0, s, a);
  } else {
    if (a.chunks > 1) {
      hipLaunchKernelGGL((recurrence_kernel<T, G, 8, 4, LOGIT, false>), dim3(a.slabs * (a.chunks - 1), rows),
                         dim3(512), 0, s, a);
      PA_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((recurrence_kernel<T, G, 8, 4, LOGIT, true>), dim3(a.slabs * a.chunks, rows), dim3(512),
                       0, s, a);
  }
  PA_LAUNCH_CHECK();
  return PA_OK;
}

template <typename T, typename G, bool LOGIT>
int run_backward(const RecArgs<T, G>& a, hipStream_t s) {
  const unsigned rows = (unsigned)(a.B < 65535 ? a.B : 65535);
  if (a.T_ <= SHORT) {
    hipLaunchKernelGGL((recurrence_grad_kernel<T, G, 1, 4, LOGIT, true>), dim3(a.slabs, rows), dim3(64), 0, s, a);
  } else {
    if (a.chunks > 1) {
      hipLaunchKernelGGL((recurrence_grad_kernel<T, G, 8, 4, LOGIT, false>), dim3(a.slabs * (a.chunks - 1), rows),
                         dim3(512), 0, s, a);
      PA_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL((recurrence_grad_kernel<T, G, 8, 4, LOGIT, true>), dim3(a.slabs * a.chunks, rows),
                       dim3(512), 0, s, a);
  }
  PA_LAUNCH_CHECK();
  return PA_OK;
}

template <typename T, typename G>
int run(const pa_recurrence_args* p, bool grad, hipStream_t s) {
  const Split sp = split_of(p->B, p->T, p->D, p->dtype);
  uint8_t* scratch = reinterpret_cast<uint8_t*>(p->scratch);
  RecArgs<T, G> a;
  a.x = reinterpret_cast<const T*>(p->x); a.x_b = p->x_b; a.x_t = p->x_t;
  a.g = reinterpret_cast<const G*>(p->gate); a.g_b = p->gate_b; a.g_t = p->gate_t;
  a.h0 = p->h0; a.resets = p->resets; a.r_b = p->resets_b; a.r_t = p->resets_t;
  a.lengths = p->lengths; a.B = p->B; a.T_ = p->T; a.D = p->D; a.reverse = p->reverse;
  a.slabs = sp.slabs; a.chunks = sp.chunks; a.chunk_tiles = sp.chunk_tiles; a.tiles = sp.tiles;
  a.agg_a = reinterpret_cast<float*>(scratch + sp.agg_a);
  a.agg_h = reinterpret_cast<float*>(scratch + sp.agg_h);
  a.agg_r = scratch + sp.agg_r;
  a.h = reinterpret_cast<T*>(p->h); a.last = p->last; a.carries = p->carries;
  a.dh = reinterpret_cast<const T*>(p->d_h); a.dh_b = p->d_h_b; a.dh_t = p->d_h_t;
  a.d_last = p->d_last;
  a.dx = reinterpret_cast<T*>(p->d_x); a.dg = reinterpret_cast<G*>(p->d_gate); a.dh0 = p->d_h0;
  if (grad)
    return p->gate_logits ? run_backward<T, G, true>(a, s) : run_backward<T, G, false>(a, s);
  return p->gate_logits ? run_forward<T, G, true>(p, a, s) : run_forward<T, G, false>(p, a, s);
}

int dispatch(const pa_recurrence_args* p, bool grad, hipStream_t s) {
  if (p->dtype == PA_F32) return run<float, float>(p, grad, s);
  if (p->dtype == PA_BF16)
    return p->gate_dtype == PA_F32 ? run<bf16_t, float>(p, grad, s) : run<bf16_t, bf16_t>(p, grad, s);
  return p->gate_dtype == PA_F32 ? run<f16_t, float>(p, grad, s) : run<f16_t, f16_t>(p, grad, s);
}

int check_args(const char* who, const pa_recurrence_args* p) {
  PA_REQUIRE(p, PA_ERR_INVALID, "%s: null argument", who);
  PA_REQUIRE(elem_size(p->dtype), PA_ERR_UNSUPPORTED, "%s: input dtype %d", who, p->dtype);
  PA_REQUIRE(p->gate_dtype == p->dtype || p->gate_dtype == PA_F32, PA_ERR_UNSUPPORTED,
             "%s: gate dtype %d with input dtype %d (the input's own, or float32)", who, p->gate_dtype, p->dtype);
  PA_REQUIRE(p->B >= 0 && p->T >= 1 && p->D >= 1 && p->D <= (1 << 24) && p->B <= (1ll << 31) / p->D, PA_ERR_INVALID,
             "%s: bad shape (batch %lld, time %lld, channels %d)", who, (long long)p->B, (long long)p->T, p->D);
  PA_REQUIRE(p->B == 0 || (p->x && p->gate), PA_ERR_INVALID, "%s: null pointer", who);
  PA_REQUIRE(p->B == 0 || p->scratch || split_of(p->B, p->T, p->D, p->dtype).bytes == 0, PA_ERR_INVALID,
             "%s: this shape needs scratch (pa_gated_recurrence_scratch)", who);
  return PA_OK;
}

}  // namespace

extern "C" int64_t pa_gated_recurrence_scratch(int64_t B, int64_t T, int32_t D, int32_t dtype) {
  return B <= 0 || T <= 0 || D <= 0 || !elem_size(dtype) ? 0 : split_of(B, T, D, dtype).bytes;
}

extern "C" int64_t pa_gated_recurrence_carries(int64_t B, int64_t T, int32_t D) {
  return B <= 0 || T <= 0 || D <= 0 ? 0 : B * ceil_div(T, tile_steps(T)) * D;
}

extern "C" int pa_gated_recurrence(const pa_recurrence_args* args, void* stream) {
  const int rc = check_args("pa_gated_recurrence", args);
  if (rc != PA_OK) return rc;
  if (args->B == 0) return PA_OK;
  PA_REQUIRE(args->h, PA_ERR_INVALID, "pa_gated_recurrence: null output");
  PA_ON_DEVICE(args->device);
  return dispatch(args, false, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int pa_gated_recurrence_grad(const pa_recurrence_args* args, void* stream) {
  const int rc = check_args("pa_gated_recurrence_grad", args);
  if (rc != PA_OK) return rc;
  if (args->B == 0) return PA_OK;
  PA_REQUIRE(args->carries && args->d_x && args->d_gate, PA_ERR_INVALID,
             "pa_gated_recurrence_grad: null pointer (carries, d_x, d_gate)");
  PA_ON_DEVICE(args->device);
  return dispatch(args, true, reinterpret_cast<hipStream_t>(stream));
}
