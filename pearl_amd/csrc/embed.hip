// Embedding of tokens and its gradient (the product one_hot(tokens) . W that pa_one_hot followed by a
// dense layer computes, without the (n, vocab) one-hot matrix):
//
//   out[i, :] = scale W[tok_i, :]          d_W[v, :] = scale sum_{i : tok_i = v} d_out[i, :]
//
// Both move rows and are bound by memory (the lookup of 16384 rows of 1024 bf16 takes 10.9 us, 5 TB/s).
// The gradient gathers instead of scattering: the tokens are
// grouped, equal tokens are summed in index order in fp32 registers, each row of d_W is rounded and
// written once; no floating-point atomics, so equal inputs give equal bits.
#include "seq_common.hpp"

using namespace pa;
using namespace pa::seq;

namespace {

// the token of row i as a row of the table; `vocab` stands for a token that has no row
template <typename I>
__device__ __forceinline__ uint32_t token_key(const I* tokens, int64_t i, uint32_t vocab) {
  const I t = tokens[i];
  return (t >= 0 && (int64_t)t < (int64_t)vocab) ? (uint32_t)t : vocab;
}

template <typename T>
struct EmbedArgs {
  const T* weight; int64_t ldw;
  uint32_t vocab; int dim;
  const void* tokens; int64_t n;
  float scale;
  T* out;
  int lane_shift;   // log2 of the lanes that share a row
};

template <typename T, typename I>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs<T> a) {
  constexpr int V = 16 / (int)sizeof(T);
  const int lanes = 1 << a.lane_shift;
  const int rows = 256 >> a.lane_shift;
  const int lane = threadIdx.x & (lanes - 1);
  const I* tokens = reinterpret_cast<const I*>(a.tokens);
  for (int64_t i = (int64_t)blockIdx.x * rows + (threadIdx.x >> a.lane_shift); i < a.n;
       i += (int64_t)gridDim.x * rows) {
    const I t = tokens[i];
    const bool has_row = t >= 0 && (int64_t)t < (int64_t)a.vocab;
    const float other = t == (I)-1 ? 0.0f : __builtin_nanf("");
    const T* src = a.weight + (has_row ? (int64_t)t * a.ldw : 0);
    T* dst = a.out + i * a.dim;
    for (int c = lane * V; c < a.dim; c += lanes * V) {
      const int left = a.dim - c;
      Pack<T, V> p;
#pragma unroll
      for (int k = 0; k < Pack<T, V>::WORDS; ++k) p.w[k] = 0;
      if (has_row) p = left >= V ? load_pack<T, V>(src + c) : load_part<T, V>(src + c, left);
      float f[V];
      unpack<T, V>(p, f);
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = has_row ? f[k] * a.scale : other;
      p = pack<T, V>(f);
      if (left >= V) store_pack<T, V>(dst + c, p);
      else store_part<T, V>(dst + c, p, left);
    }
  }
}

// ---- gradient ------------------------------------------------------------------------------------
// Grouping equal tokens, in index order, in one launch and without a pass over the batch per digit:
// workgroup w owns the tokens v with v mod W = w (neighbouring tokens, often alike in frequency, go to
// different workgroups) and reads the whole list twice from L2.  First it counts its tokens, per wave
// and token, and the tokens of the workgroups before it, which is where its part of the order begins;
// then every wave walks its sixteenth of the list again and puts each token at its place.  A token that
// fills the list costs one ballot per 64 entries like any other, so skew does not matter.  The blocks
// behind clear d_W meanwhile.  16384 tokens and 64 MB of d_W: 18.5 us (the clearing alone 11, the
// grouping alone 16; with 256 owners instead of 128 21.7: too few CUs are left to clear).
constexpr int BINS = 512;     // tokens per workgroup
constexpr int GROUP_WAVES = 16;
constexpr int AHEAD = 16;     // tokens read at once by a lane

struct GroupArgs {
  const void* tokens; int64_t n;
  uint32_t vocab;
  int owners, owner_shift;            // W, a power of two
  uint32_t* perm; uint32_t* keys;     // grouped: index and token of place p
  uint32_t* placed;                   // how many tokens have a row
  uint8_t* clear; int64_t clear_bytes;
};

template <typename I>
__global__ __launch_bounds__(1024) void group_kernel(GroupArgs a) {
  __shared__ uint32_t count[BINS * GROUP_WAVES];     // [token][wave]
  __shared__ uint32_t wave_sum[GROUP_WAVES], wave_before[GROUP_WAVES], wave_all[GROUP_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x >= a.owners) {
    typedef uint32_t U __attribute__((ext_vector_type(4), aligned(2)));
    U zero = {0, 0, 0, 0};
    const int64_t step = (int64_t)(gridDim.x - a.owners) * 1024 * 16;
    for (int64_t o = ((int64_t)(blockIdx.x - a.owners) * 1024 + tid) * 16; o < a.clear_bytes; o += step) {
      if (o + 16 <= a.clear_bytes)
        *reinterpret_cast<U*>(a.clear + o) = zero;
      else
        for (int64_t k = o; k < a.clear_bytes; ++k) a.clear[k] = 0;
    }
    return;
  }
  const I* tokens = reinterpret_cast<const I*>(a.tokens);
  const uint32_t me = blockIdx.x, low = (uint32_t)a.owners - 1;
  for (int k = tid; k < BINS * GROUP_WAVES; k += 1024) count[k] = 0;
  __syncthreads();
  // each wave's part of the list, in whole groups of 64
  const int64_t part = (a.n + 64 * GROUP_WAVES - 1) / (64 * GROUP_WAVES) * 64;
  const int64_t i0 = wave * part, i1 = i0 + part < a.n ? i0 + part : a.n;
  uint32_t before = 0, all = 0;
  uint32_t key[AHEAD];
  for (int64_t g = i0; g < i1; g += 64 * AHEAD) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int64_t i = g + 64 * u + lane;
      key[u] = i < i1 ? token_key(tokens, i, a.vocab) : a.vocab;
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const bool valid = key[u] < a.vocab;
      before += valid && (key[u] & low) < me;
      all += valid;
      if (valid && (key[u] & low) == me) atomicAdd(&count[(key[u] >> a.owner_shift) * GROUP_WAVES + wave], 1u);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    before += __shfl_xor(before, o);
    all += __shfl_xor(all, o);
  }
  if (lane == 0) {
    wave_before[wave] = before;
    wave_all[wave] = all;
  }
  __syncthreads();
  // counts -> places: exclusive sums in the order (token, wave), from this workgroup's first place on
  uint32_t sum = 0, c[GROUP_WAVES];
  if (tid < BINS) {
#pragma unroll
    for (int w = 0; w < GROUP_WAVES; ++w) {
      c[w] = count[tid * GROUP_WAVES + w];
      sum += c[w];
    }
  }
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const uint32_t y = __shfl_up(incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 63) wave_sum[wave] = incl;
  __syncthreads();
  uint32_t place = incl - sum, total = 0;
  for (int w = 0; w < GROUP_WAVES; ++w) {
    place += wave_before[w] + (w < wave ? wave_sum[w] : 0);
    total += wave_all[w];
  }
  if (me == 0 && tid == 0) *a.placed = total;
  if (tid < BINS) {
#pragma unroll
    for (int w = 0; w < GROUP_WAVES; ++w) {
      count[tid * GROUP_WAVES + w] = place;
      place += c[w];
    }
  }
  __syncthreads();
  for (int64_t g = i0; g < i1; g += 64 * AHEAD) {
    if (i1 - i0 > 64 * AHEAD) {       // up to 16384 tokens they are still in registers
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int64_t i = g + 64 * u + lane;
        key[u] = i < i1 ? token_key(tokens, i, a.vocab) : a.vocab;
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      uint64_t mine = __ballot(key[u] < a.vocab && (key[u] & low) == me);
      while (mine) {
        const int first = __ffsll((unsigned long long)mine) - 1;
        const uint32_t k = __shfl(key[u], first);
        const uint64_t same = __ballot(key[u] == k);
        uint32_t at = 0;          // this wave's own counter of the token
        if (lane == first) at = atomicAdd(&count[(k >> a.owner_shift) * GROUP_WAVES + wave], (uint32_t)__popcll(same));
        at = __shfl(at, first);
        if (key[u] == k) {
          const uint32_t p = at + __popcll(same & ((1ull << lane) - 1));
          a.perm[p] = (uint32_t)(g + 64 * u + lane);
          a.keys[p] = k;
        }
        mine &= ~same;
      }
    }
  }
}

// The places are cut into chunks of equal length, whatever the tokens: a token that is drawn often is
// summed by many chunks, a few of which share a workgroup.  A run of equal tokens that lies inside a
// chunk is rounded and written there.  The parts of one that passes a border are joined in order, in
// fp32: inside a workgroup through LDS, between workgroups through `head` (a part that began before
// this workgroup) and `tail` (one that began here and goes on) by join_kernel.  16384 rows of 1024 bf16
// in 12.4 us, 4.5 TB/s; the rows of a chunk are loaded eight at a time.
template <typename T>
struct SumArgs {
  const T* d_out; int64_t ldd;
  int dim;
  uint32_t vocab;
  int64_t n;            // places there is room for
  int64_t groups;       // workgroups along the places
  int chunk, subs;      // places per chunk, chunks per workgroup
  int lane_shift;       // log2 of the lanes that share a chunk
  const uint32_t* perm; const uint32_t* keys; const uint32_t* placed;
  float* head; float* tail;   // [groups][dim]
  float scale;
  T* d_weight;
};

template <typename T, int V>
__device__ __forceinline__ void write_row(const SumArgs<T>& a, uint32_t key, int c, const float (&acc)[V]) {
  float f[V];
#pragma unroll
  for (int k = 0; k < V; ++k) f[k] = acc[k] * a.scale;
  const Pack<T, V> p = pack<T, V>(f);
  T* dst = a.d_weight + (int64_t)key * a.dim + c;
  const int left = a.dim - c;
  if (left >= V) store_pack<T, V>(dst, p);
  else store_part<T, V>(dst, p, left);
}

template <int V>
__device__ __forceinline__ void write_partial(float* dst, int left, const float (&acc)[V]) {
  if (left >= V) store_pack<float, V>(dst, pack<float, V>(acc));
  else store_part<float, V>(dst, pack<float, V>(acc), left);
}
template <int V>
__device__ __forceinline__ void read_partial(const float* src, int left, float (&acc)[V]) {
  unpack<float, V>(left >= V ? load_pack<float, V>(src) : load_part<float, V>(src, left), acc);
}

constexpr int MAX_CHUNK = 32, MAX_SUBS = 64;

template <typename T>
__global__ __launch_bounds__(512) void sum_kernel(SumArgs<T> a) {
  constexpr int V = 16 / (int)sizeof(T), AHEAD = 8;
  extern __shared__ __attribute__((aligned(16))) float parts[];   // [2][threads][V]: heads, tails
  __shared__ uint32_t keys[MAX_CHUNK * MAX_SUBS + 2], perm[MAX_CHUNK * MAX_SUBS];
  const int lanes = 1 << a.lane_shift, threads = blockDim.x;
  const int sub = threadIdx.x >> a.lane_shift, lane = threadIdx.x & (lanes - 1);
  const int c = (int)(blockIdx.y * 256 + lane) * V;
  const int left = a.dim - c;
  const int64_t n = *a.placed;
  const int span = a.subs * a.chunk;
  const int64_t w0 = (int64_t)blockIdx.x * span;
  // keys[1 + k]: place w0 + k; one more at both ends, `vocab` where the list has none.  What lies behind
  // the n places that are taken is read (there is room) and not used: the loads need not wait for n.
  for (int k = threadIdx.x; k < span + 2; k += threads) {
    const int64_t p = w0 + k - 1;
    const uint32_t key = p >= 0 && p < a.n ? a.keys[p] : a.vocab;
    const uint32_t index = k < span && w0 + k < a.n ? a.perm[w0 + k] : 0;
    keys[k] = p < n ? key : a.vocab;
    if (k < span) perm[k] = index;
  }
  if (w0 >= n) return;
  const int here = (int)(w0 + span < n ? span : n - w0);
  __syncthreads();
  const int p0 = sub * a.chunk, p1 = p0 + a.chunk < here ? p0 + a.chunk : here;
  if (p0 < p1 && left > 0) {
    bool inside = keys[p0] != keys[p0 + 1];     // the run being summed began in this chunk
    uint32_t run = keys[p0 + 1];
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    for (int q = p0; q < p1; q += AHEAD) {
      Pack<T, V> g[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (q + u >= p1) break;
        const T* src = a.d_out + (int64_t)perm[q + u] * a.ldd + c;
        g[u] = left >= V ? load_pack<T, V>(src) : load_part<T, V>(src, left);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (q + u >= p1) break;
        const uint32_t key = keys[q + u + 1];
        if (key != run) {
          if (inside) write_row<T, V>(a, run, c, acc);
          else
#pragma unroll
            for (int k = 0; k < V; ++k) parts[threadIdx.x * V + k] = acc[k];
          inside = true;
          run = key;
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] = 0.0f;
        }
        float f[V];
        unpack<T, V>(g[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += f[k];
      }
    }
    if (inside && keys[p1 + 1] != run) write_row<T, V>(a, run, c, acc);
    else
#pragma unroll
      for (int k = 0; k < V; ++k) parts[((inside ? threads : 0) + threadIdx.x) * V + k] = acc[k];
  }
  __syncthreads();
  if (sub || left <= 0) return;
  // the chunks' open ends, in order
  float acc[V];
  bool open = keys[0] == keys[1], began_here = false;   // a run is being joined; it began in this workgroup
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;
  for (int s = 0; s < a.subs; ++s) {
    const int b0 = s * a.chunk;
    if (b0 >= here) break;
    const int b1 = b0 + a.chunk < here ? b0 + a.chunk : here;
    const uint32_t first = keys[b0 + 1], last = keys[b1];
    if (keys[b0] == first) {
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += parts[((s << a.lane_shift) + lane) * V + k];
      if (first != last || keys[b1 + 1] != last) {      // the run ends in this chunk
        if (began_here) write_row<T, V>(a, first, c, acc);
        else write_partial<V>(a.head + (int64_t)blockIdx.x * a.dim + c, left, acc);
        open = false;
      }
    }
    if (keys[b1 + 1] == last && (keys[b0] != first || first != last)) {   // one begins here and goes on
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] = parts[(threads + (s << a.lane_shift) + lane) * V + k];
      open = began_here = true;
    }
  }
  if (open) write_partial<V>((began_here ? a.tail : a.head) + (int64_t)blockIdx.x * a.dim + c, left, acc);
}

// One workgroup for each run that goes on behind the workgroup it began in: its tail, then the heads
// of those it reaches, shared by the subgroups in contiguous parts.  4 us, its chain of loads: all keys
// that decide are read at once, the parts in 16-byte loads (element by element it took 11 us).
template <typename T>
__global__ __launch_bounds__(512) void join_kernel(SumArgs<T> a) {
  constexpr int V = 16 / (int)sizeof(T), AHEAD = 8;
  extern __shared__ __attribute__((aligned(16))) float parts[];   // [threads][V]
  const int64_t span = (int64_t)a.subs * a.chunk, w0 = blockIdx.x * span, w1 = w0 + span;
  // all that decides is loaded at once: the keys around both ends of this workgroup's places, and the
  // first keys of the next 64 workgroups
  const int64_t n = *a.placed;
  const int64_t next = (blockIdx.x + 1 + (int64_t)(threadIdx.x & 63)) * span;
  const uint32_t next_key = a.keys[next < a.n ? next : 0];
  const uint32_t before = a.keys[w0 > 0 ? w0 - 1 : 0], first = a.keys[w0];
  const uint32_t run = a.keys[w1 - 1 < a.n ? w1 - 1 : 0], behind = a.keys[w1 < a.n ? w1 : 0];
  if (w1 >= n || behind != run) return;                       // ends here
  if (first == run && w0 > 0 && before == run) return;        // began before
  const int lanes = 1 << a.lane_shift;
  const int sub = threadIdx.x >> a.lane_shift, lane = threadIdx.x & (lanes - 1);
  const int c = (int)(blockIdx.y * 256 + lane) * V;
  const int left = a.dim - c < V ? a.dim - c : V;
  // how many of the next workgroups the run reaches
  int64_t reach = 0;
  uint64_t other = __ballot(!(next < n && next_key == run));
  while (!other) {
    reach += 64;
    const int64_t p = next + reach * span;
    other = __ballot(!(p < n && a.keys[p < n ? p : 0] == run));
  }
  reach += __ffsll((unsigned long long)other) - 1;
  const int64_t share = (reach + a.subs - 1) / a.subs;
  const int64_t h0 = blockIdx.x + 1 + sub * share;
  const int64_t h1 = h0 + share < blockIdx.x + 1 + reach ? h0 + share : blockIdx.x + 1 + reach;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;
  if (sub == 0) read_partial<V>(a.tail + (int64_t)blockIdx.x * a.dim + c, left, acc);
  for (int64_t h = h0; h < h1; h += AHEAD) {
    float f[AHEAD][V];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (h + u < h1) read_partial<V>(a.head + (h + u) * a.dim + c, left, f[u]);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (h + u < h1)
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += f[u][k];
  }
#pragma unroll
  for (int k = 0; k < V; ++k) parts[threadIdx.x * V + k] = acc[k];
  __syncthreads();
  if (sub || left <= 0) return;
  for (int s = 1; s < a.subs && s * share < reach; ++s)
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += parts[((s << a.lane_shift) + lane) * V + k];
  write_row<T, V>(a, run, c, acc);
}

int lane_shift_of(int dim, int v) {
  int s = 0;
  while (s < 8 && ((int64_t)v << s) < dim) ++s;
  return s;
}

struct GradLayout {
  int64_t placed, perm, keys, head, tail, bytes;
  int lane_shift, subs, chunk;
  int64_t groups;
};
// Eight chunks per workgroup (narrow rows: more, for whole waves; wide ones: 512 threads), of a length that gives the card's
// 256 CUs a workgroup each.
GradLayout grad_layout(int64_t n, int dim, int dtype) {
  GradLayout l;
  const int v = 16 / elem_size(dtype);
  l.lane_shift = lane_shift_of(dim, v);
  l.subs = 8;
  while ((l.subs << l.lane_shift) < 64) l.subs *= 2;
  while ((l.subs << l.lane_shift) > 512) l.subs /= 2;
  l.chunk = 2;
  if (n <= (int64_t)l.subs * MAX_CHUNK && n * dim * elem_size(dtype) <= 16 * 1024) {
    // so little that one workgroup sums it all, which saves the launch that joins (50 x 128 bf16, a call with
    // its lookup: 20.4 us, in many workgroups 23.1; 256 x 100: 30.5 and 22.9)
    while (n > (int64_t)l.chunk * l.subs) l.chunk *= 2;
  }
  while (l.chunk < MAX_CHUNK && n > (int64_t)l.chunk * l.subs * 256) l.chunk *= 2;
  l.groups = ceil_div(n, (int64_t)l.chunk * l.subs);
  l.placed = 0;
  l.perm = 256;
  l.keys = l.perm + round_up(n * 4, 256);
  l.head = l.keys + round_up(n * 4, 256);
  l.tail = l.head + round_up(l.groups * dim * 4, 256);
  l.bytes = l.tail + round_up(l.groups * dim * 4, 256);
  return l;
}

template <typename T>
int embed_launch(const EmbedArgs<T>& a, int token_dtype, hipStream_t s) {
  const int64_t blocks = ceil_div(a.n, 256 >> a.lane_shift);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  if (token_dtype == PA_I64) hipLaunchKernelGGL((embed_kernel<T, int64_t>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((embed_kernel<T, int32_t>), grid, dim3(256), 0, s, a);
  PA_LAUNCH_CHECK();
  return PA_OK;
}

template <typename T>
int embed_run(const void* weight, int64_t ldw, int64_t vocab, int32_t dim, const void* tokens,
              int32_t token_dtype, int64_t n, float scale, void* out, hipStream_t s) {
  EmbedArgs<T> a;
  a.weight = reinterpret_cast<const T*>(weight); a.ldw = ldw;
  a.vocab = (uint32_t)vocab; a.dim = dim; a.tokens = tokens; a.n = n; a.scale = scale;
  a.out = reinterpret_cast<T*>(out);
  a.lane_shift = lane_shift_of(dim, 16 / (int)sizeof(T));
  return embed_launch<T>(a, token_dtype, s);
}

template <typename T>
int grad_run(const void* d_out, int64_t ldd, const void* tokens, int32_t token_dtype, int64_t n,
             float scale, int64_t vocab, int32_t dim, int32_t dtype, void* d_weight, uint8_t* scratch,
             hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const GradLayout l = grad_layout(n, dim, dtype);
  GroupArgs r;
  r.tokens = tokens; r.n = n; r.vocab = (uint32_t)vocab;
  r.owners = n ? 128 : 0; r.owner_shift = 7;    // the other CUs clear meanwhile
  while (n && (int64_t)BINS << r.owner_shift < vocab) {
    r.owners *= 2;
    ++r.owner_shift;
  }
  r.perm = reinterpret_cast<uint32_t*>(scratch + l.perm);
  r.keys = reinterpret_cast<uint32_t*>(scratch + l.keys);
  r.placed = reinterpret_cast<uint32_t*>(scratch + l.placed);
  r.clear = reinterpret_cast<uint8_t*>(d_weight);
  r.clear_bytes = vocab * dim * (int64_t)sizeof(T);
  int64_t clear_blocks = ceil_div(r.clear_bytes, 1024 * 16 * 4);
  if (clear_blocks > 1024) clear_blocks = 1024;
  const dim3 group_grid((unsigned)(r.owners + clear_blocks));
  if (token_dtype == PA_I64) hipLaunchKernelGGL((group_kernel<int64_t>), group_grid, dim3(1024), 0, s, r);
  else hipLaunchKernelGGL((group_kernel<int32_t>), group_grid, dim3(1024), 0, s, r);
  PA_LAUNCH_CHECK();
  if (n == 0) return PA_OK;
  SumArgs<T> a;
  a.d_out = reinterpret_cast<const T*>(d_out); a.ldd = ldd; a.dim = dim; a.vocab = (uint32_t)vocab;
  a.n = n; a.groups = l.groups; a.chunk = l.chunk; a.subs = l.subs; a.lane_shift = l.lane_shift;
  a.perm = r.perm; a.keys = r.keys; a.placed = r.placed;
  a.head = reinterpret_cast<float*>(scratch + l.head);
  a.tail = reinterpret_cast<float*>(scratch + l.tail);
  a.scale = scale; a.d_weight = reinterpret_cast<T*>(d_weight);
  const dim3 grid((unsigned)l.groups, (unsigned)ceil_div(dim, 256 * V));
  const int threads = l.subs << l.lane_shift;
  hipLaunchKernelGGL((sum_kernel<T>), grid, dim3(threads), 2 * threads * V * 4, s, a);
  PA_LAUNCH_CHECK();
  if (l.groups > 1) {
    hipLaunchKernelGGL((join_kernel<T>), grid, dim3(threads), threads * V * 4, s, a);
    PA_LAUNCH_CHECK();
  }
  return PA_OK;
}

}  // namespace

extern "C" int pa_embed_tokens(const void* weight, int32_t dtype, int64_t ldw, int64_t vocab, int32_t dim,
                               const void* tokens, int32_t token_dtype, int64_t n, float scale, void* out,
                               int32_t device, void* stream) {
  PA_REQUIRE(elem_size(dtype), PA_ERR_UNSUPPORTED, "pa_embed_tokens: weight dtype %d", dtype);
  PA_REQUIRE(token_dtype == PA_I64 || token_dtype == PA_I32, PA_ERR_UNSUPPORTED,
             "pa_embed_tokens: token dtype %d", token_dtype);
  PA_REQUIRE(n >= 0 && dim > 0 && vocab > 0 && vocab < 0xffffffffll && ldw >= dim, PA_ERR_INVALID,
             "pa_embed_tokens: bad shape (n %lld, vocab %lld, dim %d, ldw %lld)", (long long)n,
             (long long)vocab, dim, (long long)ldw);
  PA_REQUIRE(dim <= (1 << 30), PA_ERR_UNSUPPORTED, "pa_embed_tokens: dim %d (up to 2^30)", dim);
  if (n == 0) return PA_OK;
  PA_REQUIRE(weight && tokens && out, PA_ERR_INVALID, "pa_embed_tokens: null pointer");
  PA_ON_DEVICE(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PA_F32) return embed_run<float>(weight, ldw, vocab, dim, tokens, token_dtype, n, scale, out, s);
  if (dtype == PA_BF16) return embed_run<bf16_t>(weight, ldw, vocab, dim, tokens, token_dtype, n, scale, out, s);
  return embed_run<f16_t>(weight, ldw, vocab, dim, tokens, token_dtype, n, scale, out, s);
}

extern "C" int64_t pa_embed_tokens_grad_scratch(int64_t n, int32_t dim, int32_t dtype) {
  return n <= 0 || dim <= 0 || !elem_size(dtype) ? 0 : grad_layout(n, dim, dtype).bytes;
}

extern "C" int pa_embed_tokens_grad(const void* d_out, int32_t dtype, int64_t ldd, const void* tokens,
                                    int32_t token_dtype, int64_t n, float scale, int64_t vocab, int32_t dim,
                                    void* d_weight, void* scratch, int32_t device, void* stream) {
  PA_REQUIRE(elem_size(dtype), PA_ERR_UNSUPPORTED, "pa_embed_tokens_grad: dtype %d", dtype);
  PA_REQUIRE(token_dtype == PA_I64 || token_dtype == PA_I32, PA_ERR_UNSUPPORTED,
             "pa_embed_tokens_grad: token dtype %d", token_dtype);
  PA_REQUIRE(n <= (1 << 26) && vocab <= (1 << 26), PA_ERR_UNSUPPORTED,
             "pa_embed_tokens_grad: %lld tokens, %lld rows (up to 2^26 of each)", (long long)n, (long long)vocab);
  // The grouping reads the token list twice per 512 rows of the table, at 6.2 TB/s (2^20 tokens and rows: 5.5 ms;
  // 2^22 and 2^20: 22 ms).  2^46 is a third of a second; 2^26 of both would hold the card for 23 s.
  PA_REQUIRE(n <= 0 || vocab <= (1ll << 46) / n, PA_ERR_UNSUPPORTED,
             "pa_embed_tokens_grad: %lld tokens times %lld rows (up to 2^46)", (long long)n, (long long)vocab);
  PA_REQUIRE(n >= 0 && dim > 0 && vocab > 0, PA_ERR_INVALID,
             "pa_embed_tokens_grad: bad shape (n %lld, vocab %lld, dim %d)", (long long)n, (long long)vocab, dim);
  // a grid has 65535 rows of 1024 or 2048 columns
  PA_REQUIRE(dim <= (1 << 25), PA_ERR_UNSUPPORTED, "pa_embed_tokens_grad: dim %d (up to 2^25)", dim);
  PA_REQUIRE(d_weight && (n == 0 || (d_out && tokens && scratch && ldd >= 0)), PA_ERR_INVALID,
             "pa_embed_tokens_grad: null pointer");
  PA_ON_DEVICE(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  uint8_t* w = reinterpret_cast<uint8_t*>(scratch);
  if (dtype == PA_F32)
    return grad_run<float>(d_out, ldd, tokens, token_dtype, n, scale, vocab, dim, dtype, d_weight, w, s);
  if (dtype == PA_BF16)
    return grad_run<bf16_t>(d_out, ldd, tokens, token_dtype, n, scale, vocab, dim, dtype, d_weight, w, s);
  return grad_run<f16_t>(d_out, ldd, tokens, token_dtype, n, scale, vocab, dim, dtype, d_weight, w, s);
}
