// Embedding lookup with a scale, and the gradient of the table.
//
//   out[n,:] = round(scale W[t_n,:])            dW[v,:] = round(scale sum over n with t_n = v, v != padding, of dout[n,:])
//
// The gradient sorts the tokens' positions by token (stable, digits of at most nine bits from the lowest), adds equal
// tokens' rows in 32 bits and writes every row of dW once.  The order of the additions depends on the tokens alone:
// results repeat bit by bit.  Bound by memory: what is met of the table and `out` once; dout and dW once.
#include <algorithm>

#include "language.cuh"

namespace blstm {

// ---------------------------------------------------------------- lookup
struct LookupParams {
  const void* weight;
  void* out;
  Tokens tokens;
  long long vocab, weight_stride;
  unsigned pieces;                  // of a row
  unsigned long long total;         // pieces of all rows
  float scale;
  int* mailbox;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const __grid_constant__ LookupParams p) {
  using V = Pack<T, VEC>;
  const unsigned long long i = (unsigned long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.total) return;
  const unsigned row = (unsigned)(i / p.pieces), c = (unsigned)(i - (unsigned long long)row * p.pieces);
  const long long t = p.tokens(row);
  V v;
  if (t >= 0 && t < p.vocab) {
    v = *reinterpret_cast<const V*>(static_cast<const T*>(p.weight) + t * p.weight_stride + (long long)c * VEC);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v.v[k] = Elem<T>::from_f(Elem<T>::to_f(v.v[k]) * p.scale);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v.v[k] = Elem<T>::from_f(__int_as_float(0x7fffffff));
    if (c == 0) report_token(p.mailbox, row, t);
  }
  static_cast<V*>(p.out)[i] = v;
}

// ---------------------------------------------------------------- sorting positions by token
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kMaxBins = 512;

struct SortParams {
  Tokens tokens;
  long long vocab, padding;
  unsigned n, tiles;
  int pass, passes, bits;           // of a digit
  const unsigned *keys_in, *pos_in; // pos_in null: the position itself
  unsigned *keys, *pos;
  unsigned* counts;                 // [passes][tiles][bins]
};

// A token's sort key: itself, or the vocabulary's size (behind all of them) where it gets no gradient.
__device__ __forceinline__ unsigned sort_key(const SortParams& p, unsigned i) {
  const long long t = p.tokens(i);
  return t < 0 || t >= p.vocab || t == p.padding ? (unsigned)p.vocab : (unsigned)t;
}

// Keys, and every tile's counts of the first digit; clears the counts of the others.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const __grid_constant__ SortParams p) {
  __shared__ unsigned hist[kMaxBins];
  const unsigned bins = 1u << p.bits, tile = blockIdx.x;
  for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) hist[b] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const unsigned i = (tile * ITEMS + j) * kSortThreads + threadIdx.x;
    if (i < p.n) {
      const unsigned k = sort_key(p, i);
      p.keys[i] = k;
      atomicAdd(&hist[k & (bins - 1)], 1u);
    }
  }
  __syncthreads();
  for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) {
    p.counts[(size_t)tile * bins + b] = hist[b];
    for (int q = 1; q < p.passes; ++q) p.counts[((size_t)q * p.tiles + tile) * bins + b] = 0;
  }
}

// One stable pass over a digit.  A block owns a tile: it adds up what the digit's counts say of the other tiles, ranks its
// own elements (warp by warp, each a run of consecutive ones) and puts them in their places; it counts the next digit in
// the tiles they have come to.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const __grid_constant__ SortParams p) {
  __shared__ unsigned hist[kSortWarps][kMaxBins];
  __shared__ unsigned sums[kSortWarps];
  const unsigned bins = 1u << p.bits, tile = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = p.pass * p.bits;
  for (unsigned b = tid; b < kSortWarps * kMaxBins; b += kSortThreads) (&hist[0][0])[b] = 0;
  __syncthreads();

  unsigned key[ITEMS], rank[ITEMS];
  const unsigned first = tile * (ITEMS * kSortThreads) + warp * (ITEMS * 32) + lane;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) key[j] = first + j * 32 < p.n ? p.keys_in[first + j * 32] : 0;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const bool in = first + j * 32 < p.n;
    const unsigned d = in ? (key[j] >> shift) & (bins - 1) : bins;
    const unsigned peers = __match_any_sync(0xffffffffu, d);
    const unsigned below = __popc(peers & ((1u << lane) - 1));
    rank[j] = in ? hist[warp][d] + below : 0;
    __syncwarp();
    if (in && below == 0) hist[warp][d] += __popc(peers);
    __syncwarp();
  }

  // counts of this digit before this tile, and in all of them
  unsigned before = 0, total = 0;
  if (tid < bins) {
    const unsigned* c = p.counts + (size_t)p.pass * p.tiles * bins + tid;
#pragma unroll 8
    for (unsigned t = 0; t < p.tiles; ++t) {
      const unsigned v = c[(size_t)t * bins];
      total += v;
      before += t < tile ? v : 0;
    }
  }
  unsigned scan = total;                       // inclusive over the digits
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= (unsigned)o) scan += v;
  }
  if (lane == 31) sums[warp] = scan;
  __syncthreads();
  if (tid < bins) {
    unsigned at = scan - total + before;
    for (unsigned w = 0; w < warp; ++w) at += sums[w];
    for (int w = 0; w < kSortWarps; ++w) {     // where every warp's elements of this digit begin
      const unsigned v = hist[w][tid];
      hist[w][tid] = at;
      at += v;
    }
  }
  __syncthreads();
  const bool more = p.pass + 1 < p.passes;
  unsigned* next = p.counts + (size_t)(p.pass + 1) * p.tiles * bins;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const unsigned i = first + j * 32;
    if (i >= p.n) continue;
    const unsigned to = hist[warp][(key[j] >> shift) & (bins - 1)] + rank[j];
    p.keys[to] = key[j];
    p.pos[to] = p.pos_in ? p.pos_in[i] : i;
    if (more) atomicAdd(&next[(size_t)(to / (ITEMS * kSortThreads)) * bins + ((key[j] >> (shift + p.bits)) & (bins - 1))], 1u);
  }
}

// ---------------------------------------------------------------- sums of equal tokens' rows
constexpr int kRun = 32;             // sorted positions that one group of threads adds up

struct SumParams {
  const void* dout;
  void* dweight;
  RowMap rows;
  const unsigned *keys, *pos;
  float* part;                       // [runs][2][width]: of a token that began in an earlier run, of one that goes on in the next
  unsigned n, vocab, runs, sum_blocks;
  unsigned width, pieces, group;     // group: threads of a run, a power of two
  float scale;
};

__device__ __forceinline__ unsigned lower_bound(const unsigned* keys, unsigned n, unsigned v) {
  unsigned lo = 0, hi = n;
  while (lo < hi) {
    const unsigned mid = (lo + hi) >> 1;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

constexpr int kZeroRows = 64;        // rows of dW that one block looks after

template <typename T, int VEC>
__global__ void __launch_bounds__(256) sum_kernel(const __grid_constant__ SumParams p) {
  using V = Pack<T, VEC>;
  __shared__ unsigned s_key[256 / 4 * kRun], s_pos[256 / 4 * kRun];
  if (blockIdx.x >= p.sum_blocks) {            // rows that no token names
    if (blockIdx.y) return;
    const unsigned v0 = (blockIdx.x - p.sum_blocks) * kZeroRows, rows = min((unsigned)kZeroRows, p.vocab - v0);
    if (threadIdx.x < rows) {
      const unsigned at = lower_bound(p.keys, p.n, v0 + threadIdx.x);
      s_key[threadIdx.x] = at < p.n && p.keys[at] == v0 + threadIdx.x;
    }
    __syncthreads();
    V z;
#pragma unroll
    for (int k = 0; k < VEC; ++k) z.v[k] = Elem<T>::from_f(0.f);
    V* d = static_cast<V*>(p.dweight) + (size_t)v0 * p.pieces;
    for (unsigned i = threadIdx.x; i < rows * p.pieces; i += 256)
      if (!s_key[i / p.pieces]) d[i] = z;
    return;
  }
  const unsigned runs_here = 256 / p.group, first = blockIdx.x * runs_here * kRun;
  for (unsigned i = threadIdx.x; i < runs_here * kRun; i += 256) {
    s_key[i] = first + i < p.n ? p.keys[first + i] : p.vocab;
    s_pos[i] = first + i < p.n ? p.pos[first + i] : 0;
  }
  __syncthreads();
  const unsigned mine = threadIdx.x / p.group, run = blockIdx.x * runs_here + mine;
  const unsigned c = blockIdx.y * 256 + threadIdx.x % p.group;
  if (c >= p.pieces || run >= p.runs) return;
  const unsigned* key = s_key + mine * kRun;
  const unsigned* pos = s_pos + mine * kRun;
  const unsigned i0 = run * kRun;
  const unsigned before = i0 ? p.keys[i0 - 1] : p.vocab, after = i0 + kRun < p.n ? p.keys[i0 + kRun] : p.vocab;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  for (int j = 0; j < kRun; ++j) {
    const unsigned t = key[j];
    if (t == p.vocab) break;
    const V v = *reinterpret_cast<const V*>(static_cast<const T*>(p.dout) + p.rows(pos[j]) + (size_t)c * VEC);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += Elem<T>::to_f(v.v[k]);
    const unsigned then = j + 1 < kRun ? key[j + 1] : after;
    if (then == t && j + 1 < kRun) continue;
    const bool began_before = t == before;
    if (began_before || then == t) {           // a part of a token's sum
      float* q = p.part + ((size_t)run * 2 + (began_before ? 0 : 1)) * p.width + (size_t)c * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) q[k] = acc[k];
    } else {
      V r;
#pragma unroll
      for (int k = 0; k < VEC; ++k) r.v[k] = Elem<T>::from_f(acc[k] * p.scale);
      static_cast<V*>(p.dweight)[(size_t)t * p.pieces + c] = r;
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  }
}

// Tokens whose positions reach over several runs: the parts in order.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ SumParams p) {
  const unsigned run = blockIdx.x, i0 = run * kRun, i1 = i0 + kRun;
  if (i1 >= p.n) return;
  const unsigned t = p.keys[i1 - 1];
  if (t == p.vocab || p.keys[i1] != t || (i0 && p.keys[i0 - 1] == t)) return;
  const unsigned last = (lower_bound(p.keys, p.n, t + 1) - 1) / kRun;
  for (unsigned c = blockIdx.y * 256 + threadIdx.x; c < p.width; c += gridDim.y * 256) {
    float acc = p.part[((size_t)run * 2 + 1) * p.width + c];
    for (unsigned r = run + 1; r <= last; ++r) acc += p.part[(size_t)r * 2 * p.width + c];
    static_cast<T*>(p.dweight)[(size_t)t * p.width + c] = Elem<T>::from_f(acc * p.scale);
  }
}

// ---------------------------------------------------------------- workspace
struct GradPlan {
  int items, passes, bits;
  unsigned tiles, runs;
  size_t keys[2], pos[2], counts, part, total;
};

static GradPlan grad_plan(int64_t n, int64_t vocab, int64_t width) {
  GradPlan g;
  // tiles of 2048 keep many SMs busy; larger ones where the counts of all tiles, which every block adds up, would get long
  g.items = n <= 65536 ? 4 : 16;
  g.tiles = (unsigned)((n + g.items * kSortThreads - 1) / (g.items * kSortThreads));
  int bits = 1;
  while (bits < 32 && (vocab >> bits) != 0) ++bits;       // keys go up to `vocab` itself
  g.passes = (bits + 8) / 9;
  g.bits = (bits + g.passes - 1) / g.passes;
  g.runs = (unsigned)((n + kRun - 1) / kRun);
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t o = at; at = round_up(at + bytes, 256); return o; };
  for (int k = 0; k < 2; ++k) { g.keys[k] = take(4 * n); g.pos[k] = take(4 * n); }
  g.counts = take(((size_t)g.passes * g.tiles << g.bits) * 4);
  g.part = take((size_t)g.runs * 2 * width * 4);
  g.total = at;
  return g;
}

static int check_embed(const blstm_embed_desc* d) {
  if (!d || !valid_dtype(d->dtype) || (d->token_bits != 32 && d->token_bits != 64) || !valid_rows(d->n0, d->n1) || d->vocab <= 0 ||
      d->vocab >= INT32_MAX || d->width <= 0 || d->width > INT32_MAX / 4)
    return BLSTM_E_INVALID_ARG;
  return BLSTM_OK;
}

static Tokens make_tokens(const blstm_embed_desc& d, const void* tokens) { return {tokens, row_map(d.n1, d.token_stride), d.token_bits == 64}; }

}  // namespace blstm

using namespace blstm;

extern "C" {

int blstm_embedding(const blstm_embed_desc* d, const void* tokens, const void* weight, void* out, void* stream) {
  if (int rc = check_embed(d)) return rc;
  const int64_t n = d->n0 * d->n1;
  if (n == 0) return BLSTM_OK;
  if (!tokens || !weight || !out) return BLSTM_E_INVALID_ARG;
  const int e = dtype_bytes(d->dtype);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(out) | (uintptr_t)(d->width * e) | (uintptr_t)(d->row_stride[0] * e);
  if (bits % e) return BLSTM_E_INVALID_ARG;
  const int piece = piece_bytes(bits, e);
  LookupParams p{weight, out, make_tokens(*d, tokens), d->vocab, d->row_stride[0], (unsigned)(d->width * e / piece), 0, d->scale, current_mailbox()};
  p.total = (unsigned long long)n * p.pieces;
  const unsigned long long grid = (p.total + 255) / 256;
  if (grid > INT32_MAX) return BLSTM_E_TOO_LARGE;
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (piece == 16) lookup_kernel<T, 16 / sizeof(T)><<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(p);
    else if (piece == 4) lookup_kernel<T, 4 / sizeof(T)><<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(p);
    else lookup_kernel<T, 1><<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}

size_t blstm_embedding_grad_workspace(const blstm_embed_desc* d) {
  if (check_embed(d)) return 0;
  return round_up(grad_plan(d->n0 * d->n1, d->vocab, d->width).total + 256, 256);
}

int blstm_embedding_grad(const blstm_embed_desc* d, const void* tokens, const void* dout, void* dweight, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (int rc = check_embed(d)) return rc;
  if (!dweight) return BLSTM_E_INVALID_ARG;
  const int e = dtype_bytes(d->dtype);
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t n = d->n0 * d->n1;
  if (n == 0) {
    BLSTM_CUDA_OK(cudaMemsetAsync(dweight, 0, (size_t)d->vocab * d->width * e, st));
    return BLSTM_OK;
  }
  if (!tokens || !dout) return BLSTM_E_INVALID_ARG;
  const GradPlan g = grad_plan(n, d->vocab, d->width);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < g.total) return BLSTM_E_WORKSPACE;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dweight) | (uintptr_t)(d->width * e) |
                         (uintptr_t)(d->row_stride[0] * e) | (uintptr_t)(d->row_stride[1] * e);
  if (bits % e) return BLSTM_E_INVALID_ARG;
  char* ws = static_cast<char*>(workspace);
  auto at = [&](size_t o) { return reinterpret_cast<unsigned*>(ws + o); };

  SortParams s{};
  s.tokens = make_tokens(*d, tokens);
  s.vocab = d->vocab; s.padding = d->padding;
  s.n = (unsigned)n; s.tiles = g.tiles;
  s.passes = g.passes; s.bits = g.bits;
  s.keys = at(g.keys[0]); s.counts = at(g.counts);
  if (g.items == 4) sort_count_kernel<4><<<g.tiles, kSortThreads, 0, st>>>(s);
  else sort_count_kernel<16><<<g.tiles, kSortThreads, 0, st>>>(s);
  BLSTM_CUDA_OK(cudaGetLastError());
  for (s.pass = 0; s.pass < g.passes; ++s.pass) {
    const int from = s.pass & 1;
    s.keys_in = at(g.keys[from]); s.pos_in = s.pass ? at(g.pos[from]) : nullptr;
    s.keys = at(g.keys[1 - from]); s.pos = at(g.pos[1 - from]);
    if (g.items == 4) sort_scatter_kernel<4><<<g.tiles, kSortThreads, 0, st>>>(s);
    else sort_scatter_kernel<16><<<g.tiles, kSortThreads, 0, st>>>(s);
    BLSTM_CUDA_OK(cudaGetLastError());
  }

  const int piece = piece_bytes(bits, e);
  SumParams p{};
  p.dout = dout; p.dweight = dweight;
  p.rows = row_map(d->n1, d->row_stride);
  p.keys = s.keys; p.pos = s.pos;
  p.part = reinterpret_cast<float*>(ws + g.part);
  p.n = (unsigned)n; p.vocab = (unsigned)d->vocab; p.runs = g.runs;
  p.width = (unsigned)d->width; p.pieces = (unsigned)(d->width * e / piece);
  p.group = 4;
  while (p.group < 256 && p.group < p.pieces) p.group *= 2;
  p.scale = d->scale;
  p.sum_blocks = (g.runs + 256 / p.group - 1) / (256 / p.group);
  const dim3 grid(p.sum_blocks + (p.vocab + kZeroRows - 1) / kZeroRows, (p.pieces + 255) / 256);
  if (grid.y > 65535) return BLSTM_E_TOO_LARGE;
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (piece == 16) sum_kernel<T, 16 / sizeof(T)><<<grid, 256, 0, st>>>(p);
    else if (piece == 4) sum_kernel<T, 4 / sizeof(T)><<<grid, 256, 0, st>>>(p);
    else sum_kernel<T, 1><<<grid, 256, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    join_kernel<T><<<dim3(g.runs, std::min((p.width + 255) / 256, 64u)), 256, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch(3 + g.passes);
    return BLSTM_OK;
  });
}

}  // extern "C"
