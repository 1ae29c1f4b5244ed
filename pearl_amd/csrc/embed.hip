// Embedding of tokens and its gradient (the product one_hot(tokens) . W that pa_one_hot followed by a
// dense layer computes, without the (n, vocab) one-hot matrix):
//
//   out[i, :] = scale W[tok_i, :]          d_W[v, :] = scale sum_{i : tok_i = v} d_out[i, :]
//
// Both move rows and are bound by memory.  The gradient gathers instead of scattering: the tokens are
// sorted, equal tokens are summed in index order in fp32 registers, each row of d_W is rounded and
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
// Sorting by counting: the place of token i among all is the number of tokens before it in the order
// (token, index), counted against every other token from LDS.  n^2 comparisons need no passes, no
// atomics and no further launches.  The launch also clears d_W: blocks behind the counting ones.
constexpr int RANK_TILE = 4096;

struct RankArgs {
  const void* tokens; int64_t n;
  uint32_t vocab;
  uint32_t* perm; uint32_t* keys;     // sorted: index and token of place p
  int rank_blocks;
  uint8_t* clear; int64_t clear_bytes;
};

template <typename I>
__global__ __launch_bounds__(1024) void rank_kernel(RankArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t tile[RANK_TILE];
  __shared__ uint32_t counts[16][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x >= a.rank_blocks) {
    typedef uint32_t U __attribute__((ext_vector_type(4), aligned(2)));
    U zero = {0, 0, 0, 0};
    const int64_t step = (int64_t)(gridDim.x - a.rank_blocks) * 1024 * 16;
    for (int64_t o = ((int64_t)(blockIdx.x - a.rank_blocks) * 1024 + tid) * 16; o < a.clear_bytes; o += step) {
      if (o + 16 <= a.clear_bytes)
        *reinterpret_cast<U*>(a.clear + o) = zero;
      else
        for (int64_t k = o; k < a.clear_bytes; ++k) a.clear[k] = 0;
    }
    return;
  }
  const I* tokens = reinterpret_cast<const I*>(a.tokens);
  const int64_t i = (int64_t)blockIdx.x * 64 + lane;
  const uint32_t key = i < a.n ? token_key(tokens, i, a.vocab) : 0xffffffffu;
  uint32_t before = 0;
  for (int64_t base = 0; base < a.n; base += RANK_TILE) {
    __syncthreads();
#pragma unroll
    for (int k = tid; k < RANK_TILE; k += 1024)
      tile[k] = base + k < a.n ? token_key(tokens, base + k, a.vocab) : 0xffffffffu;
    __syncthreads();
    // each wave counts a 16th of the tile, in groups of 64 that lie before, behind or at this block
#pragma unroll 1
    for (int g = wave * (RANK_TILE / 16 / 64); g < (wave + 1) * (RANK_TILE / 16 / 64); ++g) {
      const int64_t group = base / 64 + g;
      if (group * 64 >= a.n) break;
      const uint4* q = reinterpret_cast<const uint4*>(tile + g * 64);
      if (group < (int64_t)blockIdx.x) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint4 t = q[k];
          before += (t.x <= key) + (t.y <= key) + (t.z <= key) + (t.w <= key);
        }
      } else if (group > (int64_t)blockIdx.x) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint4 t = q[k];
          before += (t.x < key) + (t.y < key) + (t.z < key) + (t.w < key);
        }
      } else {
        for (int k = 0; k < 64; ++k) {
          const uint32_t t = tile[g * 64 + k];
          before += t < key || (t == key && k < lane);
        }
      }
    }
  }
  counts[wave][lane] = before;
  __syncthreads();
  if (wave == 0 && i < a.n) {
    uint32_t place = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) place += counts[w][lane];
    a.perm[place] = (uint32_t)i;
    a.keys[place] = key;
  }
}

// The sorted places are cut into chunks of equal length, whatever the tokens: a token that is drawn
// often is summed by many chunks.  A run of equal tokens that lies inside a chunk is rounded and
// written there; the parts of one that passes a border go to `head` (it began before this chunk) and
// `tail` (it began here and goes on), in fp32, and join_kernel adds them in order.
template <typename T>
struct SumArgs {
  const T* d_out; int64_t ldd;
  int dim;
  uint32_t vocab;
  int64_t n, chunks;
  int chunk;        // places per chunk
  int lane_shift;   // log2 of the lanes that share a chunk
  const uint32_t* perm; const uint32_t* keys;
  float* head; float* tail;   // [chunks][dim]
  float scale;
  T* d_weight;
};

template <typename T, int V>
__device__ __forceinline__ void write_row(const SumArgs<T>& a, uint32_t key, int c, const float (&acc)[V]) {
  if (key >= a.vocab) return;
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
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (k < left) dst[k] = acc[k];
}

template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(SumArgs<T> a) {
  constexpr int V = 16 / (int)sizeof(T);
  const int lanes = 1 << a.lane_shift;
  const int64_t chunk = (int64_t)blockIdx.x * (256 >> a.lane_shift) + (threadIdx.x >> a.lane_shift);
  const int c = (int)(blockIdx.y * 256 + (threadIdx.x & (lanes - 1))) * V;
  if (chunk >= a.chunks || c >= a.dim) return;
  const int left = a.dim - c;
  const int64_t p0 = chunk * a.chunk;
  const int64_t p1 = p0 + a.chunk < a.n ? p0 + a.chunk : a.n;
  bool inside = p0 == 0 || a.keys[p0 - 1] != a.keys[p0];   // the run being summed began in this chunk
  uint32_t run = a.keys[p0];
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;
  for (int64_t p = p0; p < p1; ++p) {
    const uint32_t key = a.keys[p];
    const T* src = a.d_out + (int64_t)a.perm[p] * a.ldd + c;
    const Pack<T, V> g = left >= V ? load_pack<T, V>(src) : load_part<T, V>(src, left);
    if (key != run) {
      if (inside) write_row<T, V>(a, run, c, acc);
      else write_partial<V>(a.head + chunk * a.dim + c, left, acc);
      inside = true;
      run = key;
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    }
    float f[V];
    unpack<T, V>(g, f);
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += f[k];
  }
  const bool goes_on = p1 < a.n && a.keys[p1] == run;
  if (!inside) write_partial<V>(a.head + chunk * a.dim + c, left, acc);
  else if (goes_on) write_partial<V>(a.tail + chunk * a.dim + c, left, acc);
  else write_row<T, V>(a, run, c, acc);
}

template <typename T>
__global__ __launch_bounds__(256) void join_kernel(SumArgs<T> a) {
  constexpr int V = 16 / (int)sizeof(T);
  const int lanes = 1 << a.lane_shift;
  const int64_t chunk = (int64_t)blockIdx.x * (256 >> a.lane_shift) + (threadIdx.x >> a.lane_shift);
  const int c = (int)(blockIdx.y * 256 + (threadIdx.x & (lanes - 1))) * V;
  if (chunk >= a.chunks || c >= a.dim) return;
  const int64_t p0 = chunk * a.chunk, p1 = p0 + a.chunk;
  if (p1 >= a.n) return;
  const uint32_t run = a.keys[p1 - 1];
  if (a.keys[p1] != run) return;                                        // ends here
  if (a.keys[p0] == run && p0 > 0 && a.keys[p0 - 1] == run) return;     // began before this chunk
  const int left = a.dim - c < V ? a.dim - c : V;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = k < left ? a.tail[chunk * a.dim + c + k] : 0.0f;
  for (int64_t d = chunk + 1; d < a.chunks && a.keys[d * a.chunk] == run; ++d) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) acc[k] += a.head[d * a.dim + c + k];
  }
  write_row<T, V>(a, run, c, acc);
}

int lane_shift_of(int dim, int v) {
  int s = 0;
  while (s < 8 && ((int64_t)v << s) < dim) ++s;
  return s;
}

// places per chunk: enough chunks to fill the card, long enough that few runs pass a border
int chunk_of(int64_t n) {
  int c = 8;
  while (c < 64 && n / c > 2048) c *= 2;
  return c;
}

struct GradLayout {
  int64_t perm, keys, head, tail, bytes;
  int chunk;
  int64_t chunks;
};
GradLayout grad_layout(int64_t n, int dim) {
  GradLayout l;
  l.chunk = chunk_of(n);
  l.chunks = ceil_div(n, l.chunk);
  l.perm = 0;
  l.keys = round_up(n * 4, 256);
  l.head = l.keys + round_up(n * 4, 256);
  l.tail = l.head + round_up(l.chunks * dim * 4, 256);
  l.bytes = l.tail + round_up(l.chunks * dim * 4, 256);
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
             float scale, int64_t vocab, int32_t dim, void* d_weight, uint8_t* scratch, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const GradLayout l = grad_layout(n, dim);
  RankArgs r;
  r.tokens = tokens; r.n = n; r.vocab = (uint32_t)vocab;
  r.perm = reinterpret_cast<uint32_t*>(scratch + l.perm);
  r.keys = reinterpret_cast<uint32_t*>(scratch + l.keys);
  r.rank_blocks = (int)ceil_div(n, 64);
  r.clear = reinterpret_cast<uint8_t*>(d_weight);
  r.clear_bytes = vocab * dim * (int64_t)sizeof(T);
  int64_t clear_blocks = ceil_div(r.clear_bytes, 1024 * 16 * 4);
  if (clear_blocks > 1024) clear_blocks = 1024;
  const dim3 rank_grid((unsigned)(r.rank_blocks + clear_blocks));
  if (token_dtype == PA_I64) hipLaunchKernelGGL((rank_kernel<int64_t>), rank_grid, dim3(1024), 0, s, r);
  else hipLaunchKernelGGL((rank_kernel<int32_t>), rank_grid, dim3(1024), 0, s, r);
  PA_LAUNCH_CHECK();
  if (n == 0) return PA_OK;
  SumArgs<T> a;
  a.d_out = reinterpret_cast<const T*>(d_out); a.ldd = ldd; a.dim = dim; a.vocab = (uint32_t)vocab;
  a.n = n; a.chunks = l.chunks; a.chunk = l.chunk;
  a.lane_shift = lane_shift_of(dim, V);
  a.perm = r.perm; a.keys = r.keys;
  a.head = reinterpret_cast<float*>(scratch + l.head);
  a.tail = reinterpret_cast<float*>(scratch + l.tail);
  a.scale = scale; a.d_weight = reinterpret_cast<T*>(d_weight);
  const dim3 grid((unsigned)ceil_div(l.chunks, 256 >> a.lane_shift), (unsigned)ceil_div(dim, 256 * V));
  hipLaunchKernelGGL((sum_kernel<T>), grid, dim3(256), 0, s, a);
  PA_LAUNCH_CHECK();
  if (l.chunks > 1) {
    hipLaunchKernelGGL((join_kernel<T>), grid, dim3(256), 0, s, a);
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
  if (n == 0) return PA_OK;
  PA_REQUIRE(weight && tokens && out, PA_ERR_INVALID, "pa_embed_tokens: null pointer");
  PA_ON_DEVICE(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PA_F32) return embed_run<float>(weight, ldw, vocab, dim, tokens, token_dtype, n, scale, out, s);
  if (dtype == PA_BF16) return embed_run<bf16_t>(weight, ldw, vocab, dim, tokens, token_dtype, n, scale, out, s);
  return embed_run<f16_t>(weight, ldw, vocab, dim, tokens, token_dtype, n, scale, out, s);
}

extern "C" int64_t pa_embed_tokens_grad_scratch(int64_t n, int32_t dim) {
  return n <= 0 || dim <= 0 ? 0 : grad_layout(n, dim).bytes;
}

extern "C" int pa_embed_tokens_grad(const void* d_out, int32_t dtype, int64_t ldd, const void* tokens,
                                    int32_t token_dtype, int64_t n, float scale, int64_t vocab, int32_t dim,
                                    void* d_weight, void* scratch, int32_t device, void* stream) {
  PA_REQUIRE(elem_size(dtype), PA_ERR_UNSUPPORTED, "pa_embed_tokens_grad: dtype %d", dtype);
  PA_REQUIRE(token_dtype == PA_I64 || token_dtype == PA_I32, PA_ERR_UNSUPPORTED,
             "pa_embed_tokens_grad: token dtype %d", token_dtype);
  PA_REQUIRE(n >= 0 && n <= (1 << 20) && dim > 0 && vocab > 0 && vocab < 0xffffffffll, PA_ERR_INVALID,
             "pa_embed_tokens_grad: bad shape (n %lld, vocab %lld, dim %d)", (long long)n, (long long)vocab, dim);
  PA_REQUIRE(d_weight && (n == 0 || (d_out && tokens && scratch && ldd >= 0)), PA_ERR_INVALID,
             "pa_embed_tokens_grad: null pointer");
  PA_ON_DEVICE(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  uint8_t* w = reinterpret_cast<uint8_t*>(scratch);
  if (dtype == PA_F32)
    return grad_run<float>(d_out, ldd, tokens, token_dtype, n, scale, vocab, dim, d_weight, w, s);
  if (dtype == PA_BF16)
    return grad_run<bf16_t>(d_out, ldd, tokens, token_dtype, n, scale, vocab, dim, d_weight, w, s);
  return grad_run<f16_t>(d_out, ldd, tokens, token_dtype, n, scale, vocab, dim, d_weight, w, s);
}
