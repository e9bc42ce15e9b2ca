// Embedding lookup with a scale, and the gradient of the table.
//
//   out[n,:] = round(scale W[t_n,:])            dW[v,:] = round(scale sum over n with t_n = v, v != padding, of dout[n,:])
//
// The gradient of many tokens sorts the tokens' positions by token (stable, digits of at most nine bits from the lowest), adds equal
// tokens' rows in 32 bits and writes every row of dW once.  The order of the additions depends on the tokens alone:
// results repeat bit by bit.  Bound by memory: what is met of the table and `out` once; dout and dW once.
#include <algorithm>

#include "language.cuh"

namespace blstm {

static_assert(sizeof(blstm_embed_desc) == 88 && sizeof(blstm_dropout_desc) == 72 && sizeof(blstm_score_desc) == 80, "as bindings lay them out");

// ---------------------------------------------------------------- lookup
struct LookupParams {
  const void* weight;
  void* out;
  Tokens tokens;
  long long vocab, weight_stride;
  unsigned n, width, pieces, group; // tokens; elements and 16-byte pieces of a row; threads side by side in a row, a power of two up to 32
  float scale;
  int* mailbox;
};

// A thread has four pieces on their way, COLS of them in a row: no divisions, which at 16 bytes a piece would take longer than
// the memory (131072 x 1024 fp16 of 131072: 85 us with them, 55 without, 95 % of the copy bandwidth).
constexpr int kLookups = 4;

template <typename T, int COLS>
__global__ void __launch_bounds__(256) lookup_kernel(const __grid_constant__ LookupParams p) {
  constexpr int N = kPer<T>, R = kLookups / COLS;
  const unsigned row0 = blockIdx.x * (256 / p.group * R) + threadIdx.x / p.group * R, c0 = blockIdx.y * (p.group * COLS) + threadIdx.x % p.group;
  long long t[R];
#pragma unroll
  for (int r = 0; r < R; ++r) t[r] = row0 + r < p.n ? p.tokens(row0 + r) : -1;
  uint4 v[R][COLS];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < COLS; ++j)
      if (t[r] >= 0 && t[r] < p.vocab && c0 + j * p.group < p.pieces)
        v[r][j] = reinterpret_cast<const uint4*>(static_cast<const T*>(p.weight) + t[r] * p.weight_stride)[c0 + j * p.group];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (row0 + r >= p.n) return;
    const bool in = t[r] >= 0 && t[r] < p.vocab;
    uint4* out = static_cast<uint4*>(p.out) + (size_t)(row0 + r) * p.pieces;
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      const unsigned c = c0 + j * p.group;
      if (c >= p.pieces) break;
      if (!in || p.scale != 1.f) {
        float z[N];
        unpack(v[r][j], z, T{});
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = in ? z[e] * p.scale : __int_as_float(0x7fffffff);
        v[r][j] = pack(z, T{});
      }
      out[c] = v[r][j];
    }
    if (!in && c0 == 0) report_token(p.mailbox, row0 + r, t[r]);
  }
}

// Rows that are no whole 16-byte pieces: a thread makes two pieces of `out`, which has no gaps, out of loads of L elements.  Bound by
// those loads (131072 x 643: fp32 95 us, bf16 80, with stores as narrow as the loads 154 and 127; 65536 x 302 bf16 27, so 24).
template <typename T, int L>
__global__ void __launch_bounds__(256) lookup_gather_kernel(const __grid_constant__ LookupParams p) {
  constexpr int N = kPer<T>, kTwo = 2;
  using V = Pack<T, L>;
  const unsigned long long total = (unsigned long long)p.n * p.width, begin = (unsigned long long)blockIdx.x * (256 * kTwo);
  alignas(16) T v[kTwo][N];
#pragma unroll
  for (int u = 0; u < kTwo; ++u) {
    const unsigned long long m = (begin + u * 256 + threadIdx.x) * N;
    if (m >= total) break;
    unsigned r = m <= 0xffffffffull ? (unsigned)m / p.width : (unsigned)(m / p.width), c = (unsigned)(m - (unsigned long long)r * p.width);
    auto known = [&](long long t) { return t >= 0 && t < p.vocab; };
    auto row = [&](long long t) { return static_cast<const T*>(p.weight) + t * p.weight_stride; };
    const T none = Elem<T>::from_f(__int_as_float(0x7fffffff));
    const long long t = p.tokens(r);
    if (!known(t) && c == 0) report_token(p.mailbox, r, t);
    if (c + N <= p.width) {
#pragma unroll
      for (int k = 0; k < N; k += L)
        if (known(t)) *reinterpret_cast<V*>(v[u] + k) = *reinterpret_cast<const V*>(row(t) + c + k);
        else
          for (int e = 0; e < L; ++e) v[u][k + e] = none;
    } else if (p.width >= N) {                 // the end of a row and the begin of the next one, or the end of all
      const bool more = r + 1 < p.n;
      const long long t2 = more ? p.tokens(r + 1) : t;
      if (more && !known(t2)) report_token(p.mailbox, r + 1, t2);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool here = c + k < p.width;
        v[u][k] = known(here ? t : t2) && m + k < total ? (here ? row(t) + c : row(t2) - (p.width - c))[k] : none;
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k, ++c) {
        if (m + k >= total) break;
        if (c == p.width) { c = 0; ++r; }
        const long long q = p.tokens(r);
        v[u][k] = known(q) ? row(q)[c] : none;
        if (!known(q) && c == 0 && k > 0) report_token(p.mailbox, r, q);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kTwo; ++u) {
    const unsigned long long m = (begin + u * 256 + threadIdx.x) * N;
    if (m >= total) break;
    T* out = static_cast<T*>(p.out) + m;
    Pack<T, N> o;
#pragma unroll
    for (int k = 0; k < N; ++k) o.v[k] = p.scale != 1.f ? Elem<T>::from_f(Elem<T>::to_f(v[u][k]) * p.scale) : v[u][k];
    if (m + N <= total && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0) *reinterpret_cast<Pack<T, N>*>(out) = o;
    else
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (m + k < total) out[k] = o.v[k];
  }
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
  char* zero;                       // what the blocks behind the tiles clear in this launch, and how much of it each
  unsigned long long zero_bytes, zero_each;
  int element;
};

// The sort is a chain of short kernels that keep few SMs busy; the others clear dW meanwhile, as much of it as that hides in
// each launch.  What is left sum_kernel clears where no token names a row.
template <int NT>
__device__ __forceinline__ void clear(const SortParams& p) {
  const unsigned long long begin = (blockIdx.x - p.tiles) * p.zero_each, end = min(p.zero_bytes, begin + p.zero_each);
  if ((reinterpret_cast<uintptr_t>(p.zero) & 15) == 0) {
    const unsigned long long whole = end & ~15ull;
    for (unsigned long long i = begin + threadIdx.x * 16; i < whole; i += NT * 16) *reinterpret_cast<uint4*>(p.zero + i) = make_uint4(0, 0, 0, 0);
    for (unsigned long long i = max(begin, whole) + threadIdx.x; i < end; i += NT) p.zero[i] = 0;
  } else if (p.element == 4) {
    for (unsigned long long i = begin + threadIdx.x * 4; i < end; i += NT * 4) *reinterpret_cast<unsigned*>(p.zero + i) = 0;
  } else {
    for (unsigned long long i = begin + threadIdx.x * 2; i < end; i += NT * 2) *reinterpret_cast<unsigned short*>(p.zero + i) = 0;
  }
}

// A token's sort key: itself, or the vocabulary's size (behind all of them) where it gets no gradient.
__device__ __forceinline__ unsigned sort_key(const SortParams& p, unsigned i) {
  const long long t = p.tokens(i);
  return t < 0 || t >= p.vocab || t == p.padding ? (unsigned)p.vocab : (unsigned)t;
}

// Keys, and every tile's counts of the first digit; clears the counts of the others.  Bound by latency, as the passes are: 4 us at
// 16384 tokens, 8 at 131072 with 32 MB cleared beside it.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const __grid_constant__ SortParams p) {
  __shared__ unsigned hist[kMaxBins];
  const unsigned bins = 1u << p.bits, tile = blockIdx.x;
  if (tile >= p.tiles) return clear<kSortThreads>(p);
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
// the tiles they have come to.  15 to 18 us at 131072 tokens with 32 MB cleared beside it.  That every block reads the counts of all
// tiles grows with their square: a pass takes 25 to 45 us at 2^20 tokens and 0.9 to 1.1 ms at 2^24, where the sums of 64 bf16 columns take 0.75.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const __grid_constant__ SortParams p) {
  __shared__ unsigned short hist[kSortWarps][kMaxBins];    // of a tile, whose numbers 16 bits hold
  __shared__ unsigned base[kMaxBins];
  __shared__ unsigned sums[kSortWarps];
  const unsigned bins = 1u << p.bits, tile = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = p.pass * p.bits;
  if (tile >= p.tiles) return clear<kSortThreads>(p);
  for (unsigned b = tid; b < kSortWarps * kMaxBins / 2; b += kSortThreads) reinterpret_cast<unsigned*>(hist)[b] = 0;
  __syncthreads();

  unsigned key[ITEMS], pos[ITEMS], rank[ITEMS];
  const unsigned first = tile * (ITEMS * kSortThreads) + warp * (ITEMS * 32) + lane;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const unsigned i = first + j * 32;
    key[j] = i < p.n ? p.keys_in[i] : 0;
    pos[j] = i < p.n && p.pos_in ? p.pos_in[i] : i;
  }

  // counts of this digit before this tile, and in all of them: a thread takes four digits of every fourth to sixty-fourth tile
  __shared__ uint4 sum_before[kSortThreads], sum_total[kSortThreads];
  {
    const unsigned quads = bins / 4, lanes = kSortThreads / quads, q = tid % quads;
    const uint4* c = reinterpret_cast<const uint4*>(p.counts + (size_t)p.pass * p.tiles * bins) + q;
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
#pragma unroll 16
    for (unsigned t = tid / quads; t < p.tiles; t += lanes) {
      const uint4 v = c[(size_t)t * quads];
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
      if (t < tile) { b.x += v.x; b.y += v.y; b.z += v.z; b.w += v.w; }
    }
    sum_total[tid] = a;
    sum_before[tid] = b;
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const bool in = first + j * 32 < p.n;
    const unsigned d = in ? (key[j] >> shift) & (bins - 1) : bins;
    const unsigned peers = __match_any_sync(0xffffffffu, d);
    const unsigned below = __popc(peers & ((1u << lane) - 1));
    rank[j] = in ? hist[warp][d] + below : 0;
    __syncwarp();
    if (in && below == 0) hist[warp][d] += (unsigned short)__popc(peers);
    __syncwarp();
  }
  __syncthreads();
  unsigned before = 0, total = 0;
  if (tid < bins)
    for (unsigned l = 0; l < kSortThreads * 4 / bins; ++l) {
      total += reinterpret_cast<const unsigned*>(sum_total)[l * bins + tid];
      before += reinterpret_cast<const unsigned*>(sum_before)[l * bins + tid];
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
    base[tid] = at;
    unsigned short in_tile = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {     // where every warp's elements of this digit begin
      const unsigned short v = hist[w][tid];
      hist[w][tid] = in_tile;
      in_tile += v;
    }
  }
  __syncthreads();
  const bool more = p.pass + 1 < p.passes;
  unsigned* next = p.counts + (size_t)(p.pass + 1) * p.tiles * bins;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const unsigned i = first + j * 32;
    if (i >= p.n) continue;
    const unsigned d = (key[j] >> shift) & (bins - 1), to = base[d] + hist[warp][d] + rank[j];
    p.keys[to] = key[j];
    p.pos[to] = pos[j];
    if (more) atomicAdd(&next[(size_t)(to / (ITEMS * kSortThreads)) * bins + ((key[j] >> (shift + p.bits)) & (bins - 1))], 1u);
  }
}

// The same sort of up to 32768 positions in one launch, by a cluster of eight blocks whose tiles are all there is: the counts of
// a digit are read from the other blocks' shared memory, and the elements change places through global memory.  17 us at 16384
// tokens with 51 MB cleared beside it, where the launches above take 19 and two launches more.
constexpr int kClusterBlocks = 8, kClusterThreads = 1024, kClusterWarps = kClusterThreads / 32;
constexpr int kClusterSort = kClusterBlocks * kClusterThreads * 4;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int ITEMS>
__global__ void __launch_bounds__(kClusterThreads) sort_cluster_kernel(const __grid_constant__ SortParams p, unsigned* keys2, unsigned* pos2) {
  __shared__ unsigned short hist[kClusterWarps][kMaxBins];
  __shared__ unsigned base[kMaxBins], count[kMaxBins];
  __shared__ unsigned sums[kClusterWarps];
  const unsigned bins = 1u << p.bits, tile = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tile >= kClusterBlocks) return clear<kClusterThreads>(p);       // (a cluster of its own)
  const unsigned first = tile * (ITEMS * kClusterThreads) + warp * (ITEMS * 32) + lane;
  unsigned key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    pos[j] = first + j * 32;
    key[j] = pos[j] < p.n ? sort_key(p, pos[j]) : 0;
  }
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    unsigned* keys = (p.passes - pass) & 1 ? p.keys : keys2;          // (the last pass ends in p.keys)
    unsigned* to_pos = (p.passes - pass) & 1 ? p.pos : pos2;
    for (unsigned b = tid; b < kClusterWarps * kMaxBins / 2; b += kClusterThreads) reinterpret_cast<unsigned*>(hist)[b] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const bool in = first + j * 32 < p.n;
      const unsigned d = in ? (key[j] >> shift) & (bins - 1) : bins;
      const unsigned peers = __match_any_sync(0xffffffffu, d);
      const unsigned below = __popc(peers & ((1u << lane) - 1));
      rank[j] = in ? hist[warp][d] + below : 0;
      __syncwarp();
      if (in && below == 0) hist[warp][d] += (unsigned short)__popc(peers);
      __syncwarp();
    }
    __syncthreads();
    if (tid < bins) {
      unsigned short in_tile = 0;
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) {
        const unsigned short v = hist[w][tid];
        hist[w][tid] = in_tile;
        in_tile += v;
      }
      count[tid] = in_tile;
    }
    cluster_sync();
    unsigned before = 0, total = 0;
    if (tid < bins) {
      const unsigned at = (unsigned)__cvta_generic_to_shared(&count[tid]);
#pragma unroll
      for (unsigned r = 0; r < kClusterBlocks; ++r) {
        unsigned remote, v;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(r));
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
        total += v;
        before += r < tile ? v : 0;
      }
    }
    unsigned scan = total;
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
      base[tid] = at;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      if (first + j * 32 >= p.n) continue;
      const unsigned d = (key[j] >> shift) & (bins - 1), to = base[d] + hist[warp][d] + rank[j];
      keys[to] = key[j];
      to_pos[to] = pos[j];
    }
    cluster_sync();                            // (also: nobody reads this block's counts any more)
    if (pass + 1 < p.passes)
#pragma unroll
      for (int j = 0; j < ITEMS; ++j)
        if (first + j * 32 < p.n) {
          key[j] = __ldcg(keys + first + j * 32);
          pos[j] = __ldcg(to_pos + first + j * 32);
        }
  }
}

// ---------------------------------------------------------------- sums of equal tokens' rows
constexpr int kMinRun = 8, kMaxRun = 64;     // sorted positions that one group of threads adds up
constexpr int kZeroRows = 16, kClearRows = 64;   // rows of dW that one block of few_kernel, of sum_kernel looks after

struct SumParams {
  const void* dout;
  void* dweight;
  RowMap rows;
  Tokens tokens;                     // (of the kernel for few tokens)
  long long padding;
  const unsigned *keys, *pos;
  float* part;                       // [runs][2][width]: of a token that began in an earlier run, of one that goes on in the next
  unsigned n, vocab, run, runs, sum_blocks;
  unsigned cleared;                  // rows of dW that the sort has cleared
  unsigned width, pieces, group;     // group: threads of a run, a power of two
  float scale;
};

// Zeros into those of the rows v0 .. v0 + rows - 1 of dW that are not `met`.
template <typename T, int VEC>
__device__ __forceinline__ void zero_rows(const SumParams& p, unsigned v0, unsigned rows, const unsigned* met) {
  using V = Pack<T, VEC>;
  V z;
#pragma unroll
  for (int k = 0; k < VEC; ++k) z.v[k] = Elem<T>::from_f(0.f);
  for (unsigned v = threadIdx.x / 32; v < rows; v += 8) {
    if (met[v]) continue;
    V* d = static_cast<V*>(p.dweight) + (size_t)(v0 + v) * p.pieces;
    for (unsigned i = threadIdx.x % 32; i < p.pieces; i += 32) d[i] = z;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void put_sum(const SumParams& p, unsigned t, unsigned c, const float (&acc)[VEC]) {
  Pack<T, VEC> r;
#pragma unroll
  for (int k = 0; k < VEC; ++k) r.v[k] = Elem<T>::from_f(acc[k] * p.scale);
  static_cast<Pack<T, VEC>*>(p.dweight)[(size_t)t * p.pieces + c] = r;
}

// What follows a position of a run: the same token, the token's last one, or its last one here of a token that goes on, or that
// began before.
enum : unsigned { kGoesOn = 0, kWhole = 1, kLastPart = 2, kFirstPart = 3 };

// A group of threads adds a run's rows up, four or eight of them on their way.  Bound by memory where there are many: 131072 x 1024 fp16 and
// 172 MB of zeros 80 to 83 us (6.2 TB/s); 16384 x 512 bf16 9 us, which are a run's latency.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) sum_kernel(const __grid_constant__ SumParams p) {
  using V = Pack<T, VEC>;
  constexpr int kRunStep = VEC * sizeof(T) == 16 ? 4 : 8;            // rows on their way at a time
  __shared__ unsigned s_key[256 / 4 * kMaxRun], s_pos[256 / 4 * kMaxRun];
  __shared__ unsigned char s_then[256 / 4 * kMaxRun];
  if (blockIdx.x >= p.sum_blocks) {            // rows that no token names
    if (blockIdx.y) return;
    const unsigned v0 = p.cleared + (blockIdx.x - p.sum_blocks) * kClearRows, rows = min((unsigned)kClearRows, p.vocab - v0);
    if (threadIdx.x < rows) {
      unsigned lo = 0, hi = p.n;
      while (lo < hi) {
        const unsigned mid = (lo + hi) >> 1;
        if (p.keys[mid] < v0 + threadIdx.x) lo = mid + 1; else hi = mid;
      }
      s_key[threadIdx.x] = lo < p.n && p.keys[lo] == v0 + threadIdx.x;
    }
    __syncthreads();
    zero_rows<T, VEC>(p, v0, rows, s_key);
    return;
  }
  const unsigned runs_here = 256 / p.group, first = blockIdx.x * runs_here * p.run;
  for (unsigned i = threadIdx.x; i < runs_here * p.run; i += 256) {
    const unsigned at = first + i, j = i % p.run;
    const unsigned t = at < p.n ? p.keys[at] : p.vocab, after = at + 1 < p.n ? p.keys[at + 1] : p.vocab;
    s_key[i] = t;
    s_pos[i] = at < p.n ? p.pos[at] : 0;
    unsigned then = kGoesOn;
    if (t != p.vocab && (after != t || j + 1 == p.run)) {
      const bool began_before = at > j && p.keys[at - j - 1] == t;
      then = began_before ? kLastPart : after == t ? kFirstPart : kWhole;
    }
    s_then[i] = (unsigned char)then;
  }
  __syncthreads();
  const unsigned mine = threadIdx.x / p.group, run = blockIdx.x * runs_here + mine;
  const unsigned c = blockIdx.y * 256 + threadIdx.x % p.group;
  if (c >= p.pieces || run >= p.runs) return;
  const unsigned* key = s_key + mine * p.run;
  const unsigned* pos = s_pos + mine * p.run;
  const unsigned char* then = s_then + mine * p.run;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  for (unsigned j0 = 0; j0 < p.run && key[j0] != p.vocab; j0 += kRunStep) {
    V v[kRunStep];
#pragma unroll
    for (int u = 0; u < kRunStep; ++u)
      if (key[j0 + u] != p.vocab) v[u] = reinterpret_cast<const V*>(static_cast<const T*>(p.dout) + p.rows(pos[j0 + u]))[c];
#pragma unroll
    for (int u = 0; u < kRunStep; ++u) {
      if (key[j0 + u] == p.vocab) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += Elem<T>::to_f(v[u].v[k]);
      const unsigned what = then[j0 + u];
      if (what == kGoesOn) continue;
      if (what == kWhole) {
        put_sum<T, VEC>(p, key[j0 + u], c, acc);
      } else {
        using Q = Pack<float, VEC % 4 ? VEC : 4>;
        Q* q = reinterpret_cast<Q*>(p.part + ((size_t)run * 2 + (what == kFirstPart)) * p.width + (size_t)c * VEC);
#pragma unroll
        for (int k = 0; k < VEC; ++k) q[k / 4].v[k % 4] = acc[k];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    }
  }
}

// Tokens whose positions reach over several runs.  A warp looks after a run, and 256 columns: where a token begins in it and
// goes on, it adds the parts up; where there are more than a few all warps of the block do, in turn (131072 tokens, the most frequent
// one 6 % of them: 10 us; with eight warps and 128 columns 22, a warp for each token 59).
constexpr unsigned kLong = 8, kJoinWarps = 16, kJoinCols = 256;

// A: 4 where rows of parts begin on 16 bytes, else 1.
template <typename T, int A>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ SumParams p) {
  using Q = Pack<float, A>;
  constexpr int K = kJoinCols / 32 / A;                    // of 32 lanes' Qs
  __shared__ float s_sum[kJoinWarps - 1][kJoinCols];
  __shared__ unsigned s_parts[kJoinWarps], s_token[kJoinWarps];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned mine = blockIdx.x * kJoinWarps + warp, end = (mine + 1) * p.run;
  unsigned t = p.vocab, parts = 0;
  if (end < p.n) {
    t = p.keys[end - 1];
    if (t != p.vocab && p.keys[end] == t && !(mine && p.keys[end - p.run - 1] == t)) {
      // the runs that it is in, 32 tried at a time, in larger steps as long as all of them are
      unsigned last = 1, step = 1;
      for (;;) {
        const unsigned k = mine + last + (lane + 1) * step;
        const unsigned hits = __popc(__ballot_sync(~0u, k < p.runs && p.keys[k * p.run] == t));
        last += hits * step;
        if (hits == 32 && step < 1024) step *= 32;
        else if (hits < 32 && step == 1) break;
        else if (hits < 32) step /= 32;
      }
      parts = last + 1;
    }
  }
  if (lane == 0) { s_parts[warp] = parts; s_token[warp] = t; }
  const unsigned q0 = blockIdx.y * (kJoinCols / A) + lane, quads = p.width / A;
  auto add = [&](unsigned run, unsigned from, unsigned parts, unsigned step, float (&acc)[K * A]) {
#pragma unroll
    for (int k = 0; k < K * A; ++k) acc[k] = 0.f;
#pragma unroll 4
    for (unsigned r = from; r < parts; r += step) {
      const Q* q = reinterpret_cast<const Q*>(p.part + ((size_t)(run + r) * 2 + (r == 0)) * p.width) + q0;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (q0 + k * 32 < quads) {
          const Q v = q[k * 32];
#pragma unroll
          for (int i = 0; i < A; ++i) acc[k * A + i] += v.v[i];
        }
    }
  };
  auto put = [&](unsigned t, const float (&acc)[K * A]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (q0 + k * 32 < quads)
#pragma unroll
        for (int i = 0; i < A; ++i) static_cast<T*>(p.dweight)[(size_t)t * p.width + (q0 + k * 32) * A + i] = Elem<T>::from_f(acc[k * A + i] * p.scale);
  };
  float acc[K * A];
  if (parts > 0 && parts <= kLong) {
    add(mine, 0, parts, 1, acc);
    put(t, acc);
  }
  __syncthreads();
  for (unsigned w = 0; w < kJoinWarps; ++w) {
    if (s_parts[w] <= kLong) continue;
    add(blockIdx.x * kJoinWarps + w, warp, s_parts[w], kJoinWarps, acc);
    if (warp)
#pragma unroll
      for (int k = 0; k < K * A; ++k) s_sum[warp - 1][k * 32 + lane] = acc[k];
    __syncthreads();
    if (warp == 0) {
      for (unsigned q = 0; q < min(s_parts[w], kJoinWarps) - 1; ++q)
#pragma unroll
        for (int k = 0; k < K * A; ++k) acc[k] += s_sum[q][k * 32 + lane];
      put(s_token[w], acc);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- few tokens: one launch, nothing sorted
// A block has a position (and a part of the columns): it looks for its token among all of them and, where it is the first
// that names it, adds the rows up, each warp some of them and then the warps in order.  Other blocks write the rows that no token names.
// 627 tokens x 301 fp32 of 10007: 8.7 us, 2 of them for 12 MB of zeros, the rest latency; the sort's launches took 18.
// 2048: a block reads all tokens, so the time grows with their square.
constexpr int kFew = 2048;

template <typename T, int VEC>
__global__ void __launch_bounds__(256) few_kernel(const __grid_constant__ SumParams p) {
  using V = Pack<T, VEC>;
  __shared__ unsigned s_met[kZeroRows];
  __shared__ unsigned s_bits[kFew / 32];
  __shared__ unsigned short s_list[kFew];
  __shared__ float s_sum[7][32][32];
  const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (blockIdx.x >= p.n) {
    if (blockIdx.y) return;
    const unsigned v0 = (blockIdx.x - p.n) * kZeroRows, rows = min((unsigned)kZeroRows, p.vocab - v0);
    if (tid < kZeroRows) s_met[tid] = 0;
    __syncthreads();
#pragma unroll 8
    for (unsigned i = tid; i < p.n; i += 256) {
      const long long t = p.tokens(i);
      if (t >= v0 && t < v0 + rows && t != p.padding) s_met[t - v0] = 1;
    }
    __syncthreads();
    zero_rows<T, VEC>(p, v0, rows, s_met);
    return;
  }
  const long long t = p.tokens(blockIdx.x);
  if (t < 0 || t >= p.vocab || t == p.padding) return;
  bool earlier = false;
  const unsigned words = (p.n + 31) / 32;
#pragma unroll 8
  for (unsigned w = warp; w < words; w += 8) {
    const unsigned i = w * 32 + lane;
    const bool same = i < p.n && p.tokens(i) == t;
    earlier |= same && i < blockIdx.x;
    const unsigned bits = __ballot_sync(~0u, same);
    if (lane == 0) s_bits[w] = bits;
  }
  if (__syncthreads_or(earlier)) return;
  // the positions in order: a word's begin behind those of the words before it
  for (unsigned w = warp; w < words; w += 8) {
    const unsigned bits = s_bits[w];
    if (bits == 0) continue;
    unsigned at = 0;
    for (unsigned q = lane; q < w; q += 32) at += __popc(s_bits[q]);
#pragma unroll
    for (int o = 16; o; o >>= 1) at += __shfl_xor_sync(~0u, at, o);
    if (bits >> lane & 1) s_list[at + __popc(bits & ((1u << lane) - 1))] = (unsigned short)(w * 32 + lane);
  }
  unsigned count = 0;
  for (unsigned w = lane; w < words; w += 32) count += __popc(s_bits[w]);
#pragma unroll
  for (int o = 16; o; o >>= 1) count += __shfl_xor_sync(~0u, count, o);
  __syncthreads();
  // a warp has every eighth of the positions and K pieces of a row in each lane
  constexpr int K = VEC == 8 ? 4 : 8;
  const unsigned c0 = blockIdx.y * (32 * K) + lane;
  float acc[K][VEC];
#pragma unroll
  for (int q = 0; q < K; ++q)
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[q][k] = 0.f;
#pragma unroll 2
  for (unsigned j = warp; j < count; j += 8) {
    const V* row = reinterpret_cast<const V*>(static_cast<const T*>(p.dout) + p.rows(s_list[j]));
    V v[K];
#pragma unroll
    for (int q = 0; q < K; ++q) if (c0 + q * 32 < p.pieces) v[q] = row[c0 + q * 32];
#pragma unroll
    for (int q = 0; q < K; ++q)
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[q][k] += c0 + q * 32 < p.pieces ? Elem<T>::to_f(v[q].v[k]) : 0.f;
  }
  if (count > 1) {
    if (warp > 0 && warp < count)
#pragma unroll
      for (int q = 0; q < K; ++q)
#pragma unroll
        for (int k = 0; k < VEC; ++k) s_sum[warp - 1][q * VEC + k][lane] = acc[q][k];
    __syncthreads();
    if (warp == 0)
      for (unsigned w = 1; w < min(count, 8u); ++w)
#pragma unroll
        for (int q = 0; q < K; ++q)
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[q][k] += s_sum[w - 1][q * VEC + k][lane];
  }
  if (warp == 0)
#pragma unroll
    for (int q = 0; q < K; ++q)
      if (c0 + q * 32 < p.pieces) put_sum<T, VEC>(p, (unsigned)t, c0 + q * 32, acc[q]);
}

// ---------------------------------------------------------------- workspace
struct GradPlan {
  int items, passes, bits;
  unsigned tiles, run, runs;
  size_t keys[2], pos[2], counts, part, total;
};

static GradPlan grad_plan(int64_t n, int64_t vocab, int64_t width) {
  GradPlan g{};
  if (n <= kFew) {
    g.total = 0;
    return g;
  }
  // tiles of 2048 keep many SMs busy; larger ones where the counts of all tiles, which every block adds up, would get long
  g.items = n <= 262144 ? 4 : 16;
  g.tiles = (unsigned)((n + g.items * kSortThreads - 1) / (g.items * kSortThreads));
  int bits = 1;
  while (bits < 32 && (vocab >> bits) != 0) ++bits;       // keys go up to `vocab` itself
  g.passes = (bits + 8) / 9;
  g.bits = std::max(2, (bits + g.passes - 1) / g.passes);
  // about 2048 runs: enough to keep all SMs busy, and no more parts to join than that takes
  g.run = kMinRun;
  while (g.run < kMaxRun && n > 2048ll * g.run) g.run *= 2;
  g.runs = (unsigned)((n + g.run - 1) / g.run);
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

static Tokens make_tokens(const blstm_embed_desc& d, const void* tokens) { return {tokens, row_map(d.n0, d.n1, d.token_stride), d.token_bits == 64}; }

}  // namespace blstm

using namespace blstm;

extern "C" {

int blstm_embedding(const blstm_embed_desc* d, const void* tokens, const void* weight, void* out, void* stream) {
  if (int rc = check_embed(d)) return rc;
  const int64_t n = d->n0 * d->n1;
  if (n == 0) return BLSTM_OK;
  if (!tokens || !weight || !out || !aligned(d->token_bits / 8, tokens)) return BLSTM_E_INVALID_ARG;
  const int e = dtype_bytes(d->dtype);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(out) | (uintptr_t)(d->width * e) | (uintptr_t)(d->row_stride[0] * e);
  if (bits % e) return BLSTM_E_INVALID_ARG;
  LookupParams p{weight, out, make_tokens(*d, tokens), d->vocab, d->row_stride[0], (unsigned)n, (unsigned)d->width, (unsigned)(d->width * e / 16), 1,
                 d->scale, current_mailbox()};
  cudaStream_t st = (cudaStream_t)stream;
  if (bits & 15u) {
    const unsigned long long blocks = ((unsigned long long)n * d->width * e + 8191) / 8192;      // of 512 pieces
    if (blocks > INT32_MAX) return BLSTM_E_TOO_LARGE;
    return with_type(d->dtype, [&](auto t) -> int {
      using T = decltype(t);
      if ((bits & 3u) == 0) lookup_gather_kernel<T, 4 / sizeof(T)><<<(unsigned)blocks, 256, 0, st>>>(p);
      else lookup_gather_kernel<T, 1><<<(unsigned)blocks, 256, 0, st>>>(p);
      BLSTM_CUDA_OK(cudaGetLastError());
      count_launch();
      return BLSTM_OK;
    });
  }
  while (p.group < 32 && p.group < p.pieces) p.group *= 2;
  const int cols = p.pieces > 64 ? 4 : p.pieces > 32 ? 2 : 1, rows = 256 / (int)p.group * (kLookups / cols);   // of a block
  const dim3 grid((unsigned)((n + rows - 1) / rows), (p.pieces + p.group * cols - 1) / (p.group * cols));
  if (grid.y > 65535) return BLSTM_E_TOO_LARGE;
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (cols == 4) lookup_kernel<T, 4><<<grid, 256, 0, st>>>(p);
    else if (cols == 2) lookup_kernel<T, 2><<<grid, 256, 0, st>>>(p);
    else lookup_kernel<T, 1><<<grid, 256, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}

size_t blstm_embedding_grad_workspace(const blstm_embed_desc* d) {
  if (check_embed(d)) return 0;
  return grad_plan(d->n0 * d->n1, d->vocab, d->width).total;
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
  if (!tokens || !dout || !aligned(d->token_bits / 8, tokens)) return BLSTM_E_INVALID_ARG;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dweight) | (uintptr_t)(d->width * e) |
                         (uintptr_t)(d->row_stride[0] * e) | (uintptr_t)(d->row_stride[1] * e);
  if (bits % e) return BLSTM_E_INVALID_ARG;
  const GradPlan g = grad_plan(n, d->vocab, d->width);
  if (g.total && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < g.total)) return BLSTM_E_WORKSPACE;
  const int piece = piece_bytes(bits, e);
  SumParams p{};
  p.dout = dout; p.dweight = dweight;
  p.rows = row_map(d->n0, d->n1, d->row_stride);
  p.tokens = make_tokens(*d, tokens); p.padding = d->padding;
  p.n = (unsigned)n; p.vocab = (unsigned)d->vocab;
  p.width = (unsigned)d->width; p.pieces = (unsigned)(d->width * e / piece);
  p.group = 4;
  while (p.group < 256 && p.group < p.pieces) p.group *= 2;
  p.scale = d->scale;
  if (n <= kFew) {
    const unsigned zero_blocks = (p.vocab + kZeroRows - 1) / kZeroRows;
    const unsigned lane_pieces = piece == 16 && e == 2 ? 4 : 8;          // (K of the kernel)
    const dim3 grid(p.n + zero_blocks, (p.pieces + 32 * lane_pieces - 1) / (32 * lane_pieces));
    if (grid.y > 65535) return BLSTM_E_TOO_LARGE;
    return with_type(d->dtype, [&](auto t) -> int {
      using T = decltype(t);
      if (piece == 16) few_kernel<T, 16 / sizeof(T)><<<grid, 256, 0, st>>>(p);
      else if (piece == 4) few_kernel<T, 4 / sizeof(T)><<<grid, 256, 0, st>>>(p);
      else few_kernel<T, 1><<<grid, 256, 0, st>>>(p);
      BLSTM_CUDA_OK(cudaGetLastError());
      count_launch();
      return BLSTM_OK;
    });
  }

  char* ws = static_cast<char*>(workspace);
  auto at = [&](size_t o) { return reinterpret_cast<unsigned*>(ws + o); };
  SortParams s{};
  s.tokens = p.tokens;
  s.vocab = d->vocab; s.padding = d->padding;
  s.n = (unsigned)n; s.tiles = g.tiles;
  s.passes = g.passes; s.bits = g.bits;
  s.keys = at(g.keys[0]); s.counts = at(g.counts);
  // dW, as much of it in each launch as the sort hides (32 MB take 5 us), 64 KB a block
  const bool cluster = n <= kClusterSort;
  const int launches = cluster ? 1 : g.passes + 1;
  const size_t row_bytes = (size_t)d->width * e;
  p.cleared = (unsigned)std::min<unsigned long long>(p.vocab, (unsigned long long)launches * (cluster ? 64u << 20 : 32u << 20) / row_bytes);
  if (bits & 15) p.cleared = p.vocab;                     // (rows in pieces of 16 bytes alone)
  const unsigned long long all = (unsigned long long)p.cleared * row_bytes, part = ((all + launches - 1) / launches + 15) & ~15ull;
  s.zero_each = 65536;
  s.element = e;
  auto blocks = [&](int launch) {
    const unsigned long long begin = std::min(all, part * launch), end = std::min(all, begin + part);
    s.zero = static_cast<char*>(dweight) + begin;
    s.zero_bytes = end - begin;
    return (unsigned)((s.zero_bytes + s.zero_each - 1) / s.zero_each);
  };
  if (cluster) {
    s.tiles = kClusterBlocks;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {kClusterBlocks, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = kClusterBlocks + (blocks(0) + kClusterBlocks - 1) / kClusterBlocks * kClusterBlocks;
    cfg.blockDim = kClusterThreads;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    s.pos = at(g.pos[0]);
    if (n <= kClusterSort / 2) BLSTM_CUDA_OK(cudaLaunchKernelEx(&cfg, sort_cluster_kernel<2>, s, at(g.keys[1]), at(g.pos[1])));
    else BLSTM_CUDA_OK(cudaLaunchKernelEx(&cfg, sort_cluster_kernel<4>, s, at(g.keys[1]), at(g.pos[1])));
  } else {
    unsigned grid = g.tiles + blocks(0);
    if (g.items == 4) sort_count_kernel<4><<<grid, kSortThreads, 0, st>>>(s);
    else sort_count_kernel<16><<<grid, kSortThreads, 0, st>>>(s);
    BLSTM_CUDA_OK(cudaGetLastError());
    for (s.pass = 0; s.pass < g.passes; ++s.pass) {
      const int from = s.pass & 1;
      s.keys_in = at(g.keys[from]); s.pos_in = s.pass ? at(g.pos[from]) : nullptr;
      s.keys = at(g.keys[1 - from]); s.pos = at(g.pos[1 - from]);
      grid = g.tiles + blocks(1 + s.pass);
      if (g.items == 4) sort_scatter_kernel<4><<<grid, kSortThreads, 0, st>>>(s);
      else sort_scatter_kernel<16><<<grid, kSortThreads, 0, st>>>(s);
      BLSTM_CUDA_OK(cudaGetLastError());
    }
  }

  p.keys = s.keys; p.pos = s.pos;
  p.part = reinterpret_cast<float*>(ws + g.part);
  p.run = g.run; p.runs = g.runs;
  p.sum_blocks = (g.runs + 256 / p.group - 1) / (256 / p.group);
  const dim3 sums(p.sum_blocks + (p.vocab - p.cleared + kClearRows - 1) / kClearRows, (p.pieces + 255) / 256), joins((g.runs + kJoinWarps - 1) / kJoinWarps, (p.width + kJoinCols - 1) / kJoinCols);
  if (sums.y > 65535 || joins.y > 65535) return BLSTM_E_TOO_LARGE;
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (piece == 16) sum_kernel<T, 16 / sizeof(T)><<<sums, 256, 0, st>>>(p);
    else if (piece == 4) sum_kernel<T, 4 / sizeof(T)><<<sums, 256, 0, st>>>(p);
    else sum_kernel<T, 1><<<sums, 256, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    if (p.width % 4 == 0) join_kernel<T, 4><<<joins, 32 * kJoinWarps, 0, st>>>(p);
    else join_kernel<T, 1><<<joins, 32 * kJoinWarps, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch(launches + 2);
    return BLSTM_OK;
  });
}

}  // extern "C"
