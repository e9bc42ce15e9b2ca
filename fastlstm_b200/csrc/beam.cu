// A step of beam search: the best continuations of every sentence's hypotheses, and the reordering of what belongs to them.
//
//   total[k,v] = score_k + z_kv - log sum_j exp z_kj       (an ended hypothesis: score_k for the end token, -inf for all others)
//   rank = total / length^penalty                          the `width` largest, equal ones by (k, v)
//
// Two launches.  The first reads every hypothesis' logits once and keeps its softmax's statistics and `width` largest logits: nothing
// else of it can be among the `width` best of the sentence.  The second joins a sentence's lists.  Bound by memory.  Totals are
// compared in 64 bits, so that what decides between two hypotheses is the sum's error alone: 2^-24 a term, 2^-22 an exponential, which
// average out to some 1e-7.
#include <algorithm>

#include "score.cuh"

namespace blstm {

struct BeamParams {
  const void* logits;
  RowMap rows;
  const float* scores;
  const uint8_t* finished;       // or null
  const long long* lengths;      // or null
  unsigned batch, beams, vocab, width, top;      // top: min(width, vocab), the length of a list
  long long end;
  double penalty;
  float2* stats;                 // [batch*beams]: largest logit, sum of exp(z - it)
  unsigned long long* keys;      // [batch*beams][top]
  float* out_scores;
  long long *parents, *tokens, *out_lengths;
  uint8_t* out_finished;
};

constexpr float kLog2E = 1.4426950408889634f;

// The launch behind this one may begin, as far as begin_behind; there it waits for all of this one.
__device__ __forceinline__ void let_begin() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void begin_behind() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A hypothesis whose logits count: it has not ended, and it is not dead.
__device__ __forceinline__ bool goes_on(const BeamParams& p, unsigned r) { return !(p.finished && p.finished[r]) && p.scores[r] != -INFINITY; }

// A part of a row: its largest logit and the sum of 2^d over it, d the distance from the reference max(m, kLowest) in powers of two.
struct alignas(8) Sum {
  float m, s;
  __device__ __forceinline__ float ref() const { return max_nan(m, kLowest); }
  __device__ __forceinline__ void rescale(float to) { s *= exp2_fast(max_nan((ref() - to) * kLog2E, kFar)); }
  __device__ __forceinline__ void join(int lanes) {
    float M = m;
    for (int o = lanes / 2; o; o >>= 1) M = max_nan(M, __shfl_xor_sync(~0u, M, o));
    rescale(max_nan(M, kLowest));
    m = M;
    for (int o = lanes / 2; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  }
};
template <int N>
__device__ __forceinline__ void take(Sum& a, const float (&z)[N]) {
  float m = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = max_nan(m, z[i]);
  if (!(m <= a.m)) {
    Sum b = a;
    a.m = max_nan(a.m, m);
    b.rescale(a.ref());
    a.s = b.s;
  }
  const float ref = a.ref();
  const Pair down = Pair::of(-ref, -ref), c = Pair::of(kLog2E, kLog2E);
  Pair s = Pair::of(a.s, 0.f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float x, y;
    ((Pair::of(z[i], z[i + 1]) + down) * c).get(x, y);
    s = s + Pair::of(exp2_fast(max_nan(x, kFar)), exp2_fast(max_nan(y, kFar)));
  }
  float s0, s1;
  s.get(s0, s1);
  a.s = s0 + s1;
}

template <typename T, int PPL>
__global__ void __launch_bounds__(32 * kWarpRows) beam_warp_kernel(const __grid_constant__ BeamParams p) {
  __shared__ unsigned long long s_cand[kWarpRows][kWarpCand];
  const unsigned warp = threadIdx.x >> 5, r = blockIdx.x * kWarpRows + warp;
  let_begin();
  if (r >= p.batch * p.beams || !goes_on(p, r)) return;
  const WarpRow<T, PPL> w(static_cast<const T*>(p.logits) + p.rows(r), p.vocab);
  Sum a{-INFINITY, 0.f};
  take(a, w.z);
  const float edge[2] = {w.edge, -INFINITY};
  take(a, edge);
  const unsigned mine = value_key(a.m);
  a.join(32);
  if (w.lane == 0) p.stats[r] = make_float2(a.m, a.s);
  warp_top(w, mine, p.top, s_cand[warp], [&](unsigned k, unsigned long long key) { p.keys[(size_t)r * p.top + k] = key; });
}

template <int NT>
struct BeamShared {
  Sum part[NT / 32];
  Sum peers[kMaxCluster];
  TopShared<NT> top;
  unsigned long long all[kMaxCluster * BLSTM_MAX_TOP];
};

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) beam_rows_kernel(const __grid_constant__ BeamParams p) {
  __shared__ BeamShared<NT> s;
  const unsigned parts = cluster_size(), part = cluster_rank(), r = blockIdx.x / parts;
  const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  let_begin();
  if (!goes_on(p, r)) return;                  // (the same for a whole cluster)
  if (parts > 1) cluster_arrive();             // this block has begun: the others may write to it
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  const Span<T> span(row, p.vocab, part, parts);
  const uint4* body = span.body();
  auto fetch = [&](unsigned i, uint4 (&v)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = i + u * NT < span.end ? load_once(body + i + u * NT) : minus_infinity(T{});
  };
  uint4 next[kUnroll];
  fetch(span.begin + tid, next);
  Sum a{-INFINITY, 0.f};
  if (tid < span.edges()) {
    const float z[2] = {ld_f(row + span.edge(tid)), -INFINITY};
    take(a, z);
  }
  for (unsigned i = span.begin + tid; i < span.end; i += kUnroll * NT) {
    float z[kUnroll * kPer<T>];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) unpack(next[u], z + u * kPer<T>, T{});
    fetch(i + kUnroll * NT, next);
    take(a, z);
  }
  const float thread_max = a.m;
  a.join(32);
  if (lane == 0) s.part[warp] = a;
  block_top(s.top, span, thread_max, p.top);
  a = s.part[lane % (NT / 32)];
  a.join(NT / 32);
  if (parts > 1) {
    cluster_wait();
    if (tid < parts) {
      static_assert(sizeof(Sum) == 8, "");
      store_to(tid, &s.peers[part], (unsigned long long)__float_as_uint(a.s) << 32 | __float_as_uint(a.m));
    }
    if (tid < parts * p.top) store_to(tid / p.top, &s.all[part * p.top + tid % p.top], s.top.best[tid % p.top]);
    cluster_arrive();
    cluster_wait();
    a = lane % kMaxCluster < parts ? s.peers[lane % kMaxCluster] : Sum{-INFINITY, 0.f};
    a.join(kMaxCluster);
    if (part == 0 && tid == 0) p.stats[r] = make_float2(a.m, a.s);
    if (tid / kMaxCluster < p.top) {
      static_assert(NT < 256 || NT == kMaxCluster * BLSTM_MAX_TOP, "clusters have blocks of 256 threads");
      const unsigned long long key = s.top.best[tid / kMaxCluster];
      const unsigned before = place_in_lists(s.all, key, parts, p.top);
      if (tid % kMaxCluster == 0 && key && before < p.top) p.keys[(size_t)r * p.top + before] = key;
    }
  } else {
    if (tid == 0) p.stats[r] = make_float2(a.m, a.s);
    if (tid < p.top) p.keys[(size_t)r * p.top + tid] = s.top.best[tid];
  }
}

// Larger ranks have larger keys, NaN the largest; no key is 0.
__device__ __forceinline__ unsigned long long rank_key(double v) {
  if (v != v) return ~0ull;
  const long long b = __double_as_longlong(v + 0.0);
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 1ull << 63;
}

constexpr int kMergeThreads = 256, kMost = BLSTM_MAX_BEAMS * BLSTM_MAX_TOP;

// A sentence's lists as one.  Every list has its `width`-th entry: what is below the largest of those is out; of what is left, eight lanes
// count what comes before an entry.
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ BeamParams p) {
  __shared__ double s_base[BLSTM_MAX_BEAMS], s_high[BLSTM_MAX_BEAMS], s_per[BLSTM_MAX_BEAMS];
  __shared__ int s_kind[BLSTM_MAX_BEAMS];      // 0 goes on, 1 has ended, 2 is dead
  __shared__ unsigned long long s_key[kMost], s_bound;
  __shared__ unsigned s_token[kMost], s_kept[kMost], s_count;
  const unsigned b = blockIdx.x, tid = threadIdx.x, total = p.beams * p.top;
  if (tid == 0) { s_bound = 0; s_count = 0; }
  if (tid < p.beams) {
    const unsigned r = b * p.beams + tid;
    const float score = p.scores[r];
    const bool ended = p.finished && p.finished[r];
    s_kind[tid] = ended ? 1 : score == -INFINITY ? 2 : 0;
    s_base[tid] = score;
    s_high[tid] = 0;
    s_per[tid] = p.penalty != 0.0 ? pow((double)(p.lengths[r] + !ended), p.penalty) : 1.0;
  }
  begin_behind();                              // (what does not need the rows' results came before)
  if (tid < p.beams && s_kind[tid] == 0) {
    const float2 st = p.stats[b * p.beams + tid];
    s_high[tid] = st.x;
    s_base[tid] = st.y == 0.f ? -INFINITY : s_base[tid] - log((double)st.y);      // (a row of nothing but -inf)
  }
  __syncthreads();
  auto total_of = [&](unsigned k, float z) { return s_base[k] == -INFINITY ? -INFINITY : s_base[k] + ((double)z - s_high[k]); };
  for (unsigned c = tid; c < total; c += kMergeThreads) {
    const unsigned k = c / p.top, i = c - k * p.top;
    unsigned token = i;
    double v = -INFINITY;
    if (s_kind[k] == 0) {
      const unsigned long long key = p.keys[(size_t)(b * p.beams + k) * p.top + i];
      token = 0xffffffffu - (unsigned)key;
      v = total_of(k, key_value((unsigned)(key >> 32)));
    } else if (s_kind[k] == 1 && s_base[k] != -INFINITY) {
      if (i == 0) { token = (unsigned)p.end; v = s_base[k]; }
      else token = i <= p.end ? i - 1 : i;
    }
    const unsigned long long key = rank_key(v / s_per[k]);
    s_key[c] = key;
    s_token[c] = token;
    if (i + 1 == p.width) atomicMax(&s_bound, key);
  }
  __syncthreads();
  const unsigned long long bound = s_bound;
  for (unsigned c = tid; c < total; c += kMergeThreads)
    if (s_key[c] >= bound) s_kept[atomicAdd(&s_count, 1u)] = c;
  __syncthreads();
  const unsigned count = s_count, lane = tid & 7;
  for (unsigned i0 = 0; i0 < count; i0 += kMergeThreads / 8) {
    const unsigned i = i0 + tid / 8;
    unsigned c = 0, before = 0;
    if (i < count) {
      c = s_kept[i];
      const unsigned long long key = s_key[c];
      const unsigned long long place = (unsigned long long)(c / p.top) << 32 | s_token[c];
      for (unsigned j = lane; j < count; j += 8) {
        const unsigned o = s_kept[j];
        const unsigned long long other = s_key[o];
        before += other > key || (other == key && ((unsigned long long)(o / p.top) << 32 | s_token[o]) < place);
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) before += __shfl_xor_sync(~0u, before, o);
    if (i < count && lane == 0 && before < p.width) {
      const unsigned k = c / p.top, token = s_token[c];
      const size_t at = (size_t)b * p.width + before;
      const unsigned r = b * p.beams + k;
      double v = -INFINITY;
      if (s_kind[k] == 0) v = total_of(k, key_value((unsigned)(p.keys[(size_t)r * p.top + (c - k * p.top)] >> 32)));
      else if (s_kind[k] == 1 && c == k * p.top) v = s_base[k];
      p.out_scores[at] = (float)v;
      p.parents[at] = k;
      p.tokens[at] = token;
      const bool ended = p.finished && p.finished[r];
      if (p.out_finished) p.out_finished[at] = ended || token == p.end;
      if (p.out_lengths) p.out_lengths[at] = p.lengths[r] + !ended;
    }
  }
}

// ---------------------------------------------------------------- reordering
// Rows are moved by groups of 1 to 32 lanes, up to kRowPieces pieces a lane; longer ones in parts.  (A thread for every piece finds its row
// by divisions: 2 x 2560 rows of 301 fp32 twice and 100 x 2560 numbers 26 us, so 8.)
constexpr int kReorderItems = 32, kReorderThreads = 256, kRowPieces = 16;
struct ReorderItem {
  const char* src;
  char* dst;
  long long outer_stride, row_stride;          // of src, in bytes
  unsigned long long units;                    // parts of rows
  unsigned per_row, parts, first;              // pieces of a row, its parts; the item's first block
  unsigned char lanes, bytes;                  // log2 of the lanes of a unit; of a piece
};
struct ReorderParams {
  ReorderItem item[kReorderItems];
  unsigned items, batch, beams, width;
  const void* parents;
  bool wide;
  int* mailbox;
};

template <typename V>
__device__ __forceinline__ void move_row(const char* src, char* dst, unsigned begin, unsigned end, unsigned lane, unsigned lanes) {
  for (unsigned i = begin + lane; i < end; i += 8 * lanes) {
    V v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      v[u] = V{};
      if (src && i + u * lanes < end) v[u] = reinterpret_cast<const V*>(src)[i + u * lanes];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * lanes < end) reinterpret_cast<V*>(dst)[i + u * lanes] = v[u];
  }
}

__device__ __forceinline__ unsigned long long quotient(unsigned long long a, unsigned b) { return a >> 32 ? a / b : (unsigned)a / b; }

__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const __grid_constant__ ReorderParams p) {
  unsigned k = 0;
  while (k + 1 < p.items && blockIdx.x >= p.item[k + 1].first) ++k;
  const ReorderItem& a = p.item[k];
  const unsigned lanes = 1u << a.lanes, lane = threadIdx.x & (lanes - 1);
  const unsigned long long unit = (unsigned long long)(blockIdx.x - a.first) * (kReorderThreads >> a.lanes) + (threadIdx.x >> a.lanes);
  if (unit >= a.units) return;
  const unsigned rows = p.batch * p.width;
  const unsigned long long out_row = a.parts == 1 ? unit : quotient(unit, a.parts), outer = quotient(out_row, rows);
  const unsigned begin = (unsigned)(unit - out_row * a.parts) * (kRowPieces << a.lanes), end = min(a.per_row, begin + (kRowPieces << a.lanes));
  const unsigned at = (unsigned)(out_row - outer * rows), b = at / p.width;
  const long long parent = p.wide ? static_cast<const long long*>(p.parents)[at] : (long long)static_cast<const int*>(p.parents)[at];
  const bool in = parent >= 0 && parent < p.beams;
  if (!in && outer == 0 && begin + lane == 0) report_token(p.mailbox, at, parent, BLSTM_E_PARENT);
  const char* src = in ? a.src + outer * a.outer_stride + ((long long)b * p.beams + parent) * a.row_stride : nullptr;
  char* dst = a.dst + out_row * a.per_row * a.bytes;
  switch (a.bytes) {
    case 16: return move_row<uint4>(src, dst, begin, end, lane, lanes);
    case 8: return move_row<uint2>(src, dst, begin, end, lane, lanes);
    case 4: return move_row<unsigned>(src, dst, begin, end, lane, lanes);
    case 2: return move_row<unsigned short>(src, dst, begin, end, lane, lanes);
    default: return move_row<unsigned char>(src, dst, begin, end, lane, lanes);
  }
}

// ---------------------------------------------------------------- host
static int check_beam(const blstm_beam_desc* d) {
  if (!d || !valid_dtype(d->dtype) || !valid_rows(d->batch, d->beams) || d->beams <= 0 || d->beams > BLSTM_MAX_BEAMS || d->width <= 0 ||
      d->width > BLSTM_MAX_TOP || d->vocab <= 0 || d->vocab >= INT32_MAX || d->width > d->beams * d->vocab || d->end_token < -1 ||
      d->end_token >= d->vocab || !(d->length_penalty >= 0 && d->length_penalty < INFINITY) || d->batch > INT32_MAX / BLSTM_MAX_TOP)
    return BLSTM_E_INVALID_ARG;
  return BLSTM_OK;
}

static unsigned list_length(const blstm_beam_desc& d) { return (unsigned)std::min<int64_t>(d.width, d.vocab); }
static size_t stats_bytes(const blstm_beam_desc& d) { return round_up((size_t)d.batch * d.beams * sizeof(float2), 256); }

// 16-byte pieces of a row: what they are at least, and at most where it does not begin on a boundary.
static unsigned beam_pieces(const BeamParams& p, size_t element) { return (unsigned)((unsigned long long)p.vocab * element / 16); }

template <typename T>
static int launch_rows(const BeamParams& p, cudaStream_t st) {
  const unsigned n = p.batch * p.beams, pieces = beam_pieces(p, sizeof(T));
  constexpr int kMostPieces = sizeof(T) == 2 ? 128 : 256;
  if (pieces <= kMostPieces) {
    const unsigned grid = (n + kWarpRows - 1) / kWarpRows, block = 32 * kWarpRows;
    if (pieces <= 32) beam_warp_kernel<T, 1><<<grid, block, 0, st>>>(p);
    else if (pieces <= 64) beam_warp_kernel<T, 2><<<grid, block, 0, st>>>(p);
    else if (pieces <= 128) beam_warp_kernel<T, 4><<<grid, block, 0, st>>>(p);
    else if constexpr (kMostPieces > 128) beam_warp_kernel<T, 8><<<grid, block, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
  } else {
    unsigned parts = 1;
    while (parts < kMaxCluster && (unsigned long long)n * parts * 2 <= 4ull * plan_sm_count() && pieces / (parts * 2) >= 256) parts *= 2;
    if ((unsigned long long)n * parts > INT32_MAX) return BLSTM_E_TOO_LARGE;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {parts, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = n * parts;
    cfg.blockDim = 256;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    BLSTM_CUDA_OK(cudaLaunchKernelEx(&cfg, beam_rows_kernel<T, 256>, p));
  }
  count_launch();
  return BLSTM_OK;
}

}  // namespace blstm

using namespace blstm;

extern "C" {

size_t blstm_beam_workspace(const blstm_beam_desc* d) {
  if (check_beam(d) || d->batch == 0) return 0;
  return round_up(stats_bytes(*d) + (size_t)d->batch * d->beams * list_length(*d) * 8, 256);
}

int blstm_beam_step(const blstm_beam_desc* d, const void* logits, const float* scores, const uint8_t* finished, const int64_t* lengths,
                    float* out_scores, int64_t* parents, int64_t* tokens, uint8_t* out_finished, int64_t* out_lengths, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (int rc = check_beam(d)) return rc;
  if (d->batch == 0) return BLSTM_OK;
  if (!logits || !scores || !out_scores || !parents || !tokens || !aligned(dtype_bytes(d->dtype), logits) || !aligned(4, scores, out_scores) ||
      !aligned(8, lengths, parents, tokens, out_lengths) || (finished && d->end_token < 0) || (d->length_penalty != 0 && !lengths) || (out_lengths && !lengths))
    return BLSTM_E_INVALID_ARG;
  if (!workspace || !aligned(256, workspace) || workspace_bytes < blstm_beam_workspace(d)) return BLSTM_E_WORKSPACE;
  BeamParams p{};
  p.logits = logits;
  p.rows = row_map(d->batch, d->beams, d->logits_stride);
  p.scores = scores; p.finished = finished;
  p.lengths = reinterpret_cast<const long long*>(lengths);
  p.batch = (unsigned)d->batch; p.beams = (unsigned)d->beams; p.vocab = (unsigned)d->vocab; p.width = (unsigned)d->width; p.top = list_length(*d);
  p.end = d->end_token;
  p.penalty = d->length_penalty;
  p.stats = static_cast<float2*>(workspace);
  p.keys = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + stats_bytes(*d));
  p.out_scores = out_scores;
  p.parents = reinterpret_cast<long long*>(parents); p.tokens = reinterpret_cast<long long*>(tokens);
  p.out_lengths = reinterpret_cast<long long*>(out_lengths);
  p.out_finished = out_finished;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = with_type(d->dtype, [&](auto t) -> int { return launch_rows<decltype(t)>(p, st); })) return rc;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = p.batch;
  cfg.blockDim = kMergeThreads;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  BLSTM_CUDA_OK(cudaLaunchKernelEx(&cfg, beam_merge_kernel, p));
  count_launch();
  return BLSTM_OK;
}

int blstm_reorder(const blstm_reorder_item* items, int n, const void* parents, int parent_bits, int64_t batch, int64_t beams, int64_t width,
                  void* stream) {
  if (n < 0 || (n && !items) || batch < 0 || beams <= 0 || width <= 0 || (batch && (beams > INT32_MAX / batch || width > INT32_MAX / batch)) ||
      (parent_bits != 32 && parent_bits != 64) || (batch && !parents) || !aligned(parent_bits / 8, parents))
    return BLSTM_E_INVALID_ARG;
  for (int k = 0; k < n; ++k)
    if (items[k].outer < 0 || items[k].inner_bytes < 0 || items[k].inner_bytes > (1ll << 36) ||
        (items[k].outer && items[k].inner_bytes && batch && (!items[k].src || !items[k].dst)))
      return BLSTM_E_INVALID_ARG;
  if (batch == 0) return BLSTM_OK;
  ReorderParams p{};
  p.batch = (unsigned)batch; p.beams = (unsigned)beams; p.width = (unsigned)width;
  p.parents = parents;
  p.wide = parent_bits == 64;
  p.mailbox = current_mailbox();
  unsigned long long blocks = 0;
  auto launch = [&]() -> int {
    if (p.items == 0) return BLSTM_OK;
    reorder_kernel<<<(unsigned)blocks, kReorderThreads, 0, (cudaStream_t)stream>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    p.items = 0;
    blocks = 0;
    return BLSTM_OK;
  };
  for (int k = 0; k < n; ++k) {
    const blstm_reorder_item& s = items[k];
    if (s.outer == 0 || s.inner_bytes == 0) continue;
    const uint64_t bits = reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst) | (uint64_t)s.inner_bytes |
                          (s.outer > 1 ? (uint64_t)s.outer_stride : 0) | (uint64_t)s.row_stride;
    const int bytes = bits & 1 ? 1 : bits & 2 ? 2 : bits & 4 ? 4 : bits & 8 ? 8 : 16;
    const uint64_t per_row = (uint64_t)s.inner_bytes / bytes, rows = (uint64_t)(batch * width);
    if (per_row > UINT32_MAX || (uint64_t)s.outer > (1ull << 48) / rows / per_row) return BLSTM_E_TOO_LARGE;
    unsigned lanes = 0;
    while (lanes < 5 && (1ull << lanes) < per_row) ++lanes;
    const uint64_t parts = (per_row + (kRowPieces << lanes) - 1) / (kRowPieces << lanes), units = (uint64_t)s.outer * rows * parts;
    const uint64_t more = (units + (kReorderThreads >> lanes) - 1) / (kReorderThreads >> lanes);
    if (more > INT32_MAX) return BLSTM_E_TOO_LARGE;
    if (p.items == kReorderItems || blocks + more > INT32_MAX)
      if (int rc = launch()) return rc;
    p.item[p.items++] = {static_cast<const char*>(s.src), static_cast<char*>(s.dst), (long long)s.outer_stride, (long long)s.row_stride, units,
                         (unsigned)per_row, (unsigned)parts, (unsigned)blocks, (unsigned char)lanes, (unsigned char)bytes};
    blocks += more;
  }
  return launch();
}

}  // extern "C"
