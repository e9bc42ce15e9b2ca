// Log probabilities of given tokens under a softmax over the vocabulary, the entropy of that distribution, and the
// likeliest tokens with theirs; and the gradient of all of them.
//
//   z = logits / temperature    lse = log sum_j exp z_j    lp_j = z_j - lse    p_j = exp lp_j
//   log_probs = lp_token        entropy = -sum_j p_j lp_j  top: the k largest logits, equal ones by their number
//   dz_j = -p_j (g + g_H (lp_j + H)) + [j = token] g_lp + sum_i [j = top_i] g_top_i,   g = g_lp + sum_i g_top_i
//
// Forward reads the logits once, backward once more and writes their gradient: bound by memory.  The softmax's statistics
// are kept in 32 bits, and a logit enters as its distance from the row's maximum, so that large common offsets cost no
// digits; distances are cut at 2^-10000, whose term is 0, so that masked logits (-inf or the type's lowest value) are finite.
#include <algorithm>

#include "language.cuh"

namespace blstm {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f, kFar = -10000.f;

struct ScoreParams {
  const void* logits;
  void* dlogits;
  RowMap rows, drows;
  Tokens tokens;
  long long ignore;
  unsigned n, vocab, parts;    // parts of a row (gradient)
  int top;
  float to_log2;               // log2(e) / temperature
  float per_temperature;       // 1 / temperature
  float *log_probs, *entropy, *top_log_probs, *stats;   // stats [3][n]: maximum, log2 of the sum, entropy
  long long* top_tokens;
  const float *g_lp, *g_h, *g_top;
  RowMap g_lp_map, g_h_map;
  int* mailbox;
};

// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The order of top alternatives: larger logits first (NaN before all), then lower numbers.  Never 0, and an order key never ~0:
// both stand for none.
__device__ __forceinline__ unsigned value_key(float z) {
  if (z != z) return 0xfffffffeu;
  const unsigned b = __float_as_uint(z + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_key(float z, unsigned j) { return (unsigned long long)value_key(z) << 32 | (0xffffffffu - j); }

__device__ __forceinline__ float key_value(unsigned key) {      // the logit of a value key (0x7ffffffe is a NaN)
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^x to 2^-22; subnormal results are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two 32-bit floats that one instruction works on.
struct Pair {
  unsigned long long v;
  __device__ __forceinline__ static Pair of(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
  }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// How many of n keys in shared memory come before `key`.
__device__ __forceinline__ unsigned rank_of(const unsigned long long* keys, unsigned n, unsigned long long key) {
  unsigned before = 0;
#pragma unroll 16
  for (unsigned q = 0; q < n; ++q) before += keys[q] > key;
  return before;
}

// A part of a row: its largest logit, and the sums of 2^d and of d 2^d over it, d the distance from the reference
// max(m, kLowest) in powers of two.
struct Part {
  float m, s, t;
  __device__ __forceinline__ float ref() const { return max_nan(m, kLowest); }
  __device__ __forceinline__ void rescale(float to, float to_log2) {      // to a reference of at least its own
    const float a = max_nan((ref() - to) * to_log2, kFar), f = exp2_fast(a);
    t = f * (t + s * a);
    s *= f;
  }
  // The whole of the parts that the 2^n lanes of a group hold, in each of them.
  __device__ __forceinline__ void join(int lanes, float to_log2) {
    float M = m;
    for (int o = lanes / 2; o; o >>= 1) M = max_nan(M, __shfl_xor_sync(~0u, M, o));
    rescale(max_nan(M, kLowest), to_log2);
    m = M;
    for (int o = lanes / 2; o; o >>= 1) {
      s += __shfl_xor_sync(~0u, s, o);
      t += __shfl_xor_sync(~0u, t, o);
    }
  }
};

// N logits into a thread's part: one comparison with the maximum so far, a rescaling where it moves.
template <int N>
__device__ __forceinline__ void take(Part& a, const float (&z)[N], float to_log2) {
  float m = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = max_nan(m, z[i]);
  if (!(m <= a.m)) {
    Part b = a;
    a.m = max_nan(a.m, m);
    b.rescale(a.ref(), to_log2);
    a.s = b.s; a.t = b.t;
  }
  const float ref = a.ref();
  const Pair down = Pair::of(-ref, -ref), c = Pair::of(to_log2, to_log2);
  Pair s = Pair::of(a.s, 0.f), t = Pair::of(a.t, 0.f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float x, y;
    ((Pair::of(z[i], z[i + 1]) + down) * c).get(x, y);
    x = max_nan(x, kFar);
    y = max_nan(y, kFar);
    const Pair e = Pair::of(exp2_fast(x), exp2_fast(y));
    s = s + e;
    t = fma2(e, Pair::of(x, y), t);
  }
  float s0, s1, t0, t1;
  s.get(s0, s1);
  t.get(t0, t1);
  a.s = s0 + s1;
  a.t = t0 + t1;
}

// What a row's statistics give.
struct Row {
  float m, log2s, entropy;
  bool none;                   // every logit is -inf
  __device__ __forceinline__ explicit Row(const Part& a) : m(a.ref()), log2s(log2f(a.s)), none(a.s == 0.f) {
    entropy = none ? 0.f : (log2s - a.t / a.s) * kLn2;
  }
  __device__ __forceinline__ float log_prob(float z, float per_temperature) const {
    return none ? -INFINITY : (z - m) * per_temperature - log2s * kLn2;
  }
};

__device__ __forceinline__ void put_row(const ScoreParams& p, unsigned r, const Row& w, long long token, float at_token) {
  const bool in = token >= 0 && token < p.vocab;
  p.log_probs[r] = in ? w.log_prob(at_token, p.per_temperature) : __int_as_float(0x7fffffff);
  p.entropy[r] = w.entropy;
  if (p.stats) {
    p.stats[r] = w.m;
    p.stats[(size_t)p.n + r] = w.log2s;
    p.stats[2 * (size_t)p.n + r] = w.entropy;
  }
  if (!in) report_token(p.mailbox, r, token);
}
__device__ __forceinline__ void put_top(const ScoreParams& p, unsigned r, const Row& w, int k, unsigned long long key) {
  p.top_log_probs[(size_t)r * p.top + k] = w.log_prob(key_value((unsigned)(key >> 32)), p.per_temperature);
  p.top_tokens[(size_t)r * p.top + k] = 0xffffffffu - (unsigned)key;
}
// A row whose token is ignored, by the threads i = 0 .. top - 1 and one at least.
__device__ __forceinline__ void put_ignored(const ScoreParams& p, unsigned r, unsigned i) {
  if (i == 0) {
    p.log_probs[r] = 0.f;
    p.entropy[r] = 0.f;
    if (p.stats)
      for (int k = 0; k < 3; ++k) p.stats[(size_t)k * p.n + r] = 0.f;
  }
  if (i < (unsigned)p.top) {
    p.top_log_probs[(size_t)r * p.top + i] = -INFINITY;
    p.top_tokens[(size_t)r * p.top + i] = -1;
  }
}

// ---------------------------------------------------------------- a row in 16-byte pieces
// What a block reads of a row: elements up to the first 16-byte boundary, pieces of 16 bytes, and the elements behind them.
template <typename T>
struct Span {
  const T* row;
  unsigned head, pieces, tail;   // of the row
  unsigned begin, end;           // this block's pieces
  bool first;                    // this block has the head and the tail
  __device__ __forceinline__ Span(const T* row, unsigned vocab, unsigned part, unsigned parts) : row(row), first(part == 0) {
    head = min(vocab, (unsigned)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (unsigned)sizeof(T));
    pieces = (vocab - head) / kPer<T>;
    tail = vocab - head - pieces * kPer<T>;
    const unsigned each = (pieces + parts - 1) / parts;
    begin = min(pieces, part * each);
    end = min(pieces, begin + each);
  }
  __device__ __forceinline__ const uint4* body() const { return reinterpret_cast<const uint4*>(row + head); }
  __device__ __forceinline__ unsigned number(unsigned piece) const { return head + piece * kPer<T>; }
  // elements of the head and the tail, in one numbering: 2 * kPer - 2 at most
  __device__ __forceinline__ unsigned edges() const { return first ? head + tail : 0; }
  __device__ __forceinline__ unsigned edge(unsigned i) const { return i < head ? i : head + pieces * kPer<T> + (i - head); }
};

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 minus_infinity(float) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
__device__ __forceinline__ uint4 minus_infinity(__nv_bfloat16) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
__device__ __forceinline__ uint4 minus_infinity(__half) { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }

// ---------------------------------------------------------------- small vocabularies: a warp has a row in its registers
// (16384 rows of 1000 fp32 logits: forward 13 us, with blocks 21, backward 22; of 1500 to 2000 bf16 forward 20, with blocks 24, but
// with 5 alternatives 77 and with blocks 47, and backward 41 where blocks take 27: so half as long for those.)
constexpr int kWarpPieces = 256, kWarpRows = 8, kWarpCand = 128;

// PPL pieces and an element of the edges in each lane.
template <typename T, int PPL>
struct WarpRow {
  Span<T> span;
  unsigned lane;
  float z[PPL * kPer<T>], edge;
  __device__ __forceinline__ WarpRow(const T* row, unsigned vocab) : span(row, vocab, 0, 1), lane(threadIdx.x & 31) {
    uint4 v[PPL];
#pragma unroll
    for (int u = 0; u < PPL; ++u) v[u] = u * 32 + lane < span.pieces ? load_once(span.body() + u * 32 + lane) : minus_infinity(T{});
    edge = lane < span.edges() ? ld_f(row + span.edge(lane)) : -INFINITY;
#pragma unroll
    for (int u = 0; u < PPL; ++u) unpack(v[u], z + u * kPer<T>, T{});
  }
  // f(logit, number) for every logit that this lane has; the lanes stay together (f may use the warp), `in` says whose are real
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int i = 0; i < PPL * kPer<T>; ++i) {
      const unsigned piece = i / kPer<T> * 32 + lane;
      f(z[i], span.number(piece) + i % kPer<T>, piece < span.pieces);
    }
    f(edge, span.edge(lane), lane < span.edges());
  }
};

template <typename T, int PPL, bool TOP>
__global__ void __launch_bounds__(32 * kWarpRows) score_warp_kernel(const __grid_constant__ ScoreParams p) {
  __shared__ unsigned long long s_cand[TOP ? kWarpRows : 1][TOP ? kWarpCand : 1];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.x * kWarpRows + warp;
  if (r >= p.n) return;
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  const long long token = p.tokens(r);
  const WarpRow<T, PPL> w(row, p.vocab);       // (before the token is there; a row that is ignored is small)
  if (token == p.ignore) {
    put_ignored(p, r, lane);
    return;
  }
  const float at_token = token >= 0 && token < p.vocab ? ld_f(row + token) : 0.f;
  Part a{-INFINITY, 0.f, 0.f};
  take(a, w.z, p.to_log2);
  const float edge[2] = {w.edge, -INFINITY};
  take(a, edge, p.to_log2);
  const unsigned mine = value_key(a.m);        // (of a lane without logits: that of -inf)
  a.join(32, p.to_log2);
  const Row stats(a);
  if (lane == 0) put_row(p, r, stats, token, at_token);
  if constexpr (TOP) {
    // The k-th largest of the lanes' maxima is a lower bound of the k-th largest logit: what is below it is out.
    unsigned left = mine, bound, found = 0;
    do {
      bound = __reduce_max_sync(~0u, left);
      found += __popc(__ballot_sync(~0u, left == bound));
      if (left == bound) left = 0;             // (no key is 0)
    } while (found < (unsigned)p.top);
    unsigned count = 0;
    w.each([&](float z, unsigned j, bool in) {
      const unsigned key = value_key(z), who = __ballot_sync(~0u, in && key >= bound);
      const unsigned at = count + __popc(who & ((1u << lane) - 1));
      if (in && key >= bound && at < kWarpCand) s_cand[warp][at] = order_key(z, j);
      count += __popc(who);
    });
    __syncwarp();
    if (count <= kWarpCand) {
      for (unsigned i = lane; i < count; i += 32) {
        const unsigned long long key = s_cand[warp][i];
        const unsigned before = rank_of(s_cand[warp], count, key);
        if (before < (unsigned)p.top) put_top(p, r, stats, (int)before, key);
      }
    } else {                                   // (many equal logits) one after the other
      unsigned long long last = ~0ull;
      for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0;
        w.each([&](float z, unsigned j, bool in) {
          const unsigned long long key = order_key(z, j);
          if (in && key < last && key > best) best = key;
        });
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
        if (lane == 0) put_top(p, r, stats, k, best);
        last = best;
      }
    }
  }
}

// ---------------------------------------------------------------- large vocabularies: a block, or a cluster of them, has a row
constexpr int kUnroll = 2, kGroups = 64, kCand = 1024, kMaxCluster = 8;

__device__ __forceinline__ unsigned cluster_size() {
  unsigned v;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(v));
  return v;
}
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned v;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(v));
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// the same variable in another block of the cluster
template <typename V>
__device__ __forceinline__ void store_to(unsigned block, V* p, unsigned long long v) {
  static_assert(sizeof(V) == 8, "");
  unsigned a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(block));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

template <int NT>
struct ScoreShared {
  Part part[NT / 32];
  uint2 peers[kMaxCluster][2];                          // maximum and sum, second sum, of every block of a cluster
  alignas(16) unsigned group[kGroups];
  unsigned owner[NT];
  unsigned least[kGroups / 32];
  unsigned owners, count;
  unsigned long long bound;
  unsigned long long cand[kCand];
  unsigned long long best[BLSTM_MAX_TOP];               // of this block
  unsigned long long all[kMaxCluster * BLSTM_MAX_TOP];  // of every block of a cluster
};

// The `top` first of a block's logits in order, into s.best: threads' maxima bound them from below, the threads whose
// maximum reaches that bound (few more than `top`) have their logits looked at again.
template <typename T, int NT>
__device__ __forceinline__ void block_top(ScoreShared<NT>& s, const Span<T>& span, float thread_max, unsigned top) {
  const unsigned tid = threadIdx.x, lane = tid & 31;
  const unsigned mine = value_key(thread_max);
  unsigned g = mine;
#pragma unroll
  for (int o = 1; o < NT / kGroups; o <<= 1) g = max(g, __shfl_xor_sync(~0u, g, o));
  if (tid % (NT / kGroups) == 0) s.group[tid / (NT / kGroups)] = g;
  if (tid == 0) { s.owners = 0; s.count = 0; }
  if (tid < top) s.best[tid] = 0;              // (a block may have fewer)
  __syncthreads();
  // the `top`-th largest of the groups' maxima: the smallest that fewer than `top` are above (equal ones count alike)
  if (tid < kGroups) {
    const unsigned g = s.group[tid];
    unsigned above = 0;
#pragma unroll 4
    for (unsigned i = 0; i < kGroups; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(s.group + i);
      above += (v.x > g) + (v.y > g) + (v.z > g) + (v.w > g);
    }
    const unsigned least = __reduce_min_sync(~0u, above < top ? g : ~0u);
    if (lane == 0) s.least[tid / 32] = least;
  }
  __syncthreads();
  const unsigned bound = min(s.least[0], s.least[1]);
  if (mine >= bound) s.owner[atomicAdd(&s.owners, 1u)] = tid;
  __syncthreads();
  auto offer = [&](float z, unsigned j, unsigned long long least) {
    const unsigned long long key = order_key(z, j);
    if (key < least) return;
    const unsigned at = atomicAdd(&s.count, 1u);
    if (at < kCand) s.cand[at] = key;
  };
  auto look = [&](const uint4& v, unsigned piece, unsigned long long least) {
    float z[kPer<T>], m;
    unpack(v, z, T{});
    m = z[0];
#pragma unroll
    for (int i = 1; i < kPer<T>; ++i) m = max_nan(m, z[i]);
    if (value_key(m) < (unsigned)(least >> 32)) return;
    unsigned some = 0;
#pragma unroll
    for (int i = 0; i < kPer<T>; ++i) some |= (value_key(z[i]) >= (unsigned)(least >> 32) ? 1u : 0u) << i;
#pragma unroll 1
    for (; some; some &= some - 1) {           // (few, so in little code: it runs once a block)
      const unsigned j = span.number(piece) + __ffs(some) - 1;
      offer(ld_f(span.row + j), j, least);
    }
  };
  // the owners' pieces, all threads side by side
  const unsigned owners = s.owners, each = (span.end - span.begin + NT - 1) / NT;
  const unsigned long long least = (unsigned long long)bound << 32;
  constexpr int kLook = 2;
  for (unsigned i0 = tid; i0 < owners * each; i0 += kLook * NT) {
    uint4 v[kLook];
    unsigned piece[kLook];
#pragma unroll
    for (int u = 0; u < kLook; ++u) {
      const unsigned i = i0 + u * NT;
      piece[u] = i < owners * each ? span.begin + s.owner[i / each] + i % each * NT : span.end;
      if (piece[u] < span.end) v[u] = span.body()[piece[u]];
    }
#pragma unroll
    for (int u = 0; u < kLook; ++u)
      if (piece[u] < span.end) look(v[u], piece[u], least);
  }
  for (unsigned i = tid; i < owners; i += NT)
    if (s.owner[i] < span.edges()) offer(ld_f(span.row + span.edge(s.owner[i])), span.edge(s.owner[i]), least);
  __syncthreads();
  while (s.count > kCand) {                    // (many equal logits) a higher bound, from some of them, until they fit
    const unsigned long long key = s.cand[tid];
    if (rank_of(s.cand, NT, key) == top - 1) s.bound = key;
    __syncthreads();
    if (tid == 0) s.count = 0;
    __syncthreads();
    const unsigned long long more = s.bound;
    for (unsigned piece = span.begin + tid; piece < span.end; piece += NT) look(span.body()[piece], piece, more);
    if (tid < span.edges()) offer(ld_f(span.row + span.edge(tid)), span.edge(tid), more);
    __syncthreads();
  }
  const unsigned count = s.count;
  for (unsigned i = tid; i < count; i += NT) {
    const unsigned long long key = s.cand[i];
    const unsigned before = rank_of(s.cand, count, key);
    if (before < top) s.best[before] = key;
  }
  __syncthreads();
}

// 8192 x 50000 bf16 130 us (6.3 TB/s; the exponentials, one a logit, at 73 % of their unit), fp32 at the copy bandwidth.  Few rows are a
// chain of latencies: 1 x 131072 4.2 us, with 20 alternatives 6.6.
template <typename T, bool TOP, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) score_kernel(const __grid_constant__ ScoreParams p) {
  __shared__ ScoreShared<NT> s;
  const unsigned parts = cluster_size(), part = cluster_rank(), r = blockIdx.x / parts;
  const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  const Span<T> span(row, p.vocab, part, parts);
  const uint4* body = span.body();
  // kUnroll pieces are on their way while those before them are added up
  auto fetch = [&](unsigned i, uint4 (&v)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = i + u * NT < span.end ? load_once(body + i + u * NT) : minus_infinity(T{});
  };
  uint4 next[kUnroll];
  const long long token = p.tokens(r);
  if (parts > 1) {                             // few rows: nothing waits for the token, not even where it is to be ignored
    fetch(span.begin + tid, next);
    cluster_arrive();                          // this block has begun: the others may write to it
  } else {
    if (token == p.ignore) {
      put_ignored(p, r, tid);
      return;
    }
    fetch(span.begin + tid, next);
  }
  Part a{-INFINITY, 0.f, 0.f};
  if (tid < span.edges()) {
    const float z[2] = {ld_f(row + span.edge(tid)), -INFINITY};
    take(a, z, p.to_log2);
  }
  for (unsigned i = span.begin + tid; i < span.end; i += kUnroll * NT) {
    float z[kUnroll * kPer<T>];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) unpack(next[u], z + u * kPer<T>, T{});
    fetch(i + kUnroll * NT, next);
    take(a, z, p.to_log2);
  }
  const float at_token = tid == 0 && part == 0 && token >= 0 && token < p.vocab ? ld_f(row + token) : 0.f;
  const float thread_max = a.m;
  a.join(32, p.to_log2);
  if (lane == 0) s.part[warp] = a;
  if constexpr (TOP) block_top(s, span, thread_max, (unsigned)p.top);
  else __syncthreads();
  a = s.part[lane % (NT / 32)];
  a.join((NT / 32), p.to_log2);
  if (parts > 1) {
    // every block tells all what its part has come to
    cluster_wait();
    if (tid < parts) {
      store_to(tid, &s.peers[part][0], (unsigned long long)__float_as_uint(a.s) << 32 | __float_as_uint(a.m));
      store_to(tid, &s.peers[part][1], __float_as_uint(a.t));
    }
    if (TOP && tid < parts * p.top) store_to(tid / p.top, &s.all[part * p.top + tid % p.top], s.best[tid % p.top]);
    cluster_arrive();
    cluster_wait();
    const unsigned q = lane % kMaxCluster;
    a = q < parts ? Part{__uint_as_float(s.peers[q][0].x), __uint_as_float(s.peers[q][0].y), __uint_as_float(s.peers[q][1].x)} : Part{-INFINITY, 0.f, 0.f};
    a.join(kMaxCluster, p.to_log2);
    if (token == p.ignore) {                   // (the same for the whole cluster)
      if (part == 0) put_ignored(p, r, tid);
      return;
    }
  }
  const Row w(a);
  if (tid == 0 && part == 0) put_row(p, r, w, token, at_token);
  if constexpr (TOP) {
    if (parts == 1) {
      if (tid < (unsigned)p.top) put_top(p, r, w, tid, s.best[tid]);
    } else if (tid / kMaxCluster < (unsigned)p.top) {
      // The blocks' lists, each in order, as one: a block has the places of its own keys, eight lanes a key, each of which finds
      // how many of one list come before it.
      static_assert(NT < 256 || NT == kMaxCluster * BLSTM_MAX_TOP, "clusters have blocks of 256 threads");
      const unsigned q = tid % kMaxCluster;
      const unsigned long long key = s.best[tid / kMaxCluster];
      unsigned before = 0;
      if (q < parts)
#pragma unroll
        for (unsigned step = BLSTM_MAX_TOP; step; step >>= 1)
          if (before + step <= (unsigned)p.top && s.all[q * p.top + before + step - 1] > key) before += step;
#pragma unroll
      for (int o = 1; o < kMaxCluster; o <<= 1) before += __shfl_xor_sync(0xffu << (lane & ~7u), before, o);
      if (q == 0 && key && before < (unsigned)p.top) put_top(p, r, w, before, key);
    }
  }
}

// ---------------------------------------------------------------- gradient
struct RowGrad {
  float m, log2s, g_lp, a, b;  // dz_j = 2^d (a + b d) and what given and top tokens add, d = log2 p_j
  long long token;
  bool zero;
  __device__ __forceinline__ RowGrad(const ScoreParams& p, unsigned r) : token(p.tokens(r)) {
    m = p.stats[r];
    log2s = p.stats[(size_t)p.n + r];
    const float h = p.stats[2 * (size_t)p.n + r];
    const bool in = token >= 0 && token < p.vocab;
    zero = token == p.ignore || !in || log2s == -INFINITY;
    g_lp = p.g_lp && in ? p.g_lp[p.g_lp_map(r)] : 0.f;
    const float g_h = p.g_h ? p.g_h[p.g_h_map(r)] : 0.f;
    float g = g_lp;
    if (p.g_top && !zero)
      for (int k = 0; k < p.top; ++k) g += p.g_top[(size_t)r * p.top + k];
    a = -(g + g_h * h) * p.per_temperature;
    b = -g_h * kLn2 * p.per_temperature;
  }
  __device__ __forceinline__ float operator()(float z, float to_log2) const {
    const float d = max_nan(fmaf(z - m, to_log2, -log2s), kFar);
    return exp2_fast(d) * fmaf(b, d, a);
  }
  // The i-th of the token (0) and the top tokens (1 .. top): its number where nobody before it has the same, else -1.
  __device__ __forceinline__ long long special(const ScoreParams& p, unsigned r, unsigned i) const {
    const long long* tops = p.top_tokens + (size_t)r * p.top;
    const long long j = i == 0 ? token : tops[i - 1];
    if (i > 0 && (p.g_top == nullptr || j == token)) return -1;
    return j >= 0 && j < p.vocab ? j : -1;
  }
  // The gradient of logit j, which is the token or a top token.
  __device__ __forceinline__ float at(const ScoreParams& p, unsigned r, float z, long long j) const {
    float extra = j == token ? g_lp : 0.f;
    if (p.g_top)
      for (int k = 0; k < p.top; ++k)
        if (p.top_tokens[(size_t)r * p.top + k] == j) extra += p.g_top[(size_t)r * p.top + k];
    return fmaf(extra, p.per_temperature, (*this)(z, p.to_log2));
  }
};

// 16384 x 205 fp32 8.2 us, x 1000 22 us (91 % of the copy bandwidth).
template <typename T, int PPL>
__global__ void __launch_bounds__(32 * kWarpRows) score_grad_warp_kernel(const __grid_constant__ ScoreParams p) {
  const unsigned lane = threadIdx.x & 31, r = blockIdx.x * kWarpRows + (threadIdx.x >> 5);
  if (r >= p.n) return;
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  T* out = static_cast<T*>(p.dlogits) + p.drows(r);
  WarpRow<T, PPL> w(row, p.vocab);
  const RowGrad g(p, r);
  auto grad = [&](float z, unsigned j) { return g.zero ? 0.f : j == g.token ? fmaf(g.g_lp, p.per_temperature, g(z, p.to_log2)) : g(z, p.to_log2); };
  uint4* body = reinterpret_cast<uint4*>(out + w.span.head);          // (the same address modulo 16 as the logits')
#pragma unroll
  for (int u = 0; u < PPL; ++u) {
    const unsigned piece = u * 32 + lane;
#pragma unroll
    for (int i = 0; i < kPer<T>; ++i) w.z[u * kPer<T> + i] = grad(w.z[u * kPer<T> + i], w.span.number(piece) + i);
    if (piece < w.span.pieces) body[piece] = pack(w.z + u * kPer<T>, T{});
  }
  if (lane < w.span.edges()) out[w.span.edge(lane)] = Elem<T>::from_f(grad(w.edge, w.span.edge(lane)));
  if (p.g_top == nullptr || g.zero) return;
  __syncwarp();                                // top tokens are written again, behind the others
  for (unsigned i = lane; i <= (unsigned)p.top; i += 32) {
    const long long j = g.special(p, r, i);
    if (j >= 0) out[j] = Elem<T>::from_f(g.at(p, r, ld_f(row + j), j));
  }
}

// A block has a part of a row, kGradPieces pieces a thread at most: blocks that run at a time write neighbouring memory (4096 x
// 50000 fp32 and 8192 x 50000 bf16 with whole rows 290 and 267 us, with 4 pieces a thread 254 and 276, with 6 248 and 265, with 8
// 248 and 269).
constexpr int kGradPieces = 6;

template <typename T, int NT>
__global__ void __launch_bounds__(NT) score_grad_kernel(const __grid_constant__ ScoreParams p) {
  const unsigned r = blockIdx.x / p.parts, part = blockIdx.x - r * p.parts, tid = threadIdx.x;
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  T* out = static_cast<T*>(p.dlogits) + p.drows(r);
  const Span<T> span(row, p.vocab, part, p.parts);
  const unsigned first = span.begin + tid;
  uint4* out_body = reinterpret_cast<uint4*>(out + span.head);        // (the same address modulo 16 as the logits')
  uint4 v[kGradPieces];
  if (p.tokens(r) != p.ignore)
#pragma unroll
    for (int u = 0; u < kGradPieces; ++u) if (first + u * NT < span.end) v[u] = load_once(span.body() + first + u * NT);
  const RowGrad g(p, r);
  if (g.zero) {
#pragma unroll
    for (int u = 0; u < kGradPieces; ++u) if (first + u * NT < span.end) out_body[first + u * NT] = make_uint4(0, 0, 0, 0);
    if (tid < span.edges()) out[span.edge(tid)] = Elem<T>::from_f(0.f);
    return;
  }
  if (tid < span.edges()) out[span.edge(tid)] = Elem<T>::from_f(g(ld_f(row + span.edge(tid)), p.to_log2));
  const Pair down = Pair::of(-g.m, -g.m), c = Pair::of(p.to_log2, p.to_log2), minus = Pair::of(-g.log2s, -g.log2s);
  const Pair a = Pair::of(g.a, g.a), b = Pair::of(g.b, g.b);
#pragma unroll
  for (int u = 0; u < kGradPieces; ++u)
    if (first + u * NT < span.end) {
      float z[kPer<T>];
      unpack(v[u], z, T{});
#pragma unroll
      for (int k = 0; k < kPer<T>; k += 2) {
        float x, y;
        fma2(Pair::of(z[k], z[k + 1]) + down, c, minus).get(x, y);
        x = max_nan(x, kFar);
        y = max_nan(y, kFar);
        (Pair::of(exp2_fast(x), exp2_fast(y)) * fma2(b, Pair::of(x, y), a)).get(z[k], z[k + 1]);
      }
      out_body[first + u * NT] = pack(z, T{});
    }
  __syncthreads();                             // the few logits that get more are written again, behind the others
  if (tid <= (p.g_top ? (unsigned)p.top : 0u)) {
    const long long j = g.special(p, r, tid);
    const bool edge = j >= 0 && (j < span.head || j >= span.head + span.pieces * kPer<T>);
    const unsigned piece = (unsigned)(j - span.head) / kPer<T>;
    if (j >= 0 && (edge ? span.first : piece >= span.begin && piece < span.end)) out[j] = Elem<T>::from_f(g.at(p, r, ld_f(row + j), j));
  }
}

static int check_score(const blstm_score_desc* d, const void* logits, const void* tokens) {
  if (!d || !valid_dtype(d->dtype) || (d->token_bits != 32 && d->token_bits != 64) || !valid_rows(d->n0, d->n1) || d->vocab <= 0 ||
      d->vocab >= INT32_MAX || d->top < 0 || d->top > BLSTM_MAX_TOP || d->top > d->vocab || !(d->temperature >= 1e-30f && d->temperature < INFINITY))
    return BLSTM_E_INVALID_ARG;
  if (d->n0 && d->n1 && (!logits || !tokens || !aligned(dtype_bytes(d->dtype), logits) || !aligned(d->token_bits / 8, tokens))) return BLSTM_E_INVALID_ARG;
  return BLSTM_OK;
}

static ScoreParams score_params(const blstm_score_desc& d, const void* logits, const void* tokens) {
  ScoreParams p{};
  p.logits = logits;
  p.rows = row_map(d.n0, d.n1, d.logits_stride);
  p.tokens = {tokens, row_map(d.n0, d.n1, d.token_stride), d.token_bits == 64};
  p.ignore = d.ignore;
  p.n = (unsigned)(d.n0 * d.n1); p.vocab = (unsigned)d.vocab; p.top = d.top;
  p.per_temperature = (float)(1.0 / d.temperature);
  p.to_log2 = (float)(1.4426950408889634 / d.temperature);
  return p;
}

// 16-byte pieces of a row: what they are at least, and at most where it does not begin on a boundary (fewer elements are left).
static unsigned row_pieces(const ScoreParams& p, size_t element) { return (unsigned)((unsigned long long)p.vocab * element / 16); }

// Threads of a block.  A row ends with some hundred clocks in which nothing is read, and the more rows an SM has at a time the
// less that shows; long rows have it seldom and take the threads.  bf16, us with 64 / 128 / 256 threads: 32768 x 10007 118 / 142 /
// 225, 8192 x 50000 130 / 132 / 139, 4096 x 131072 175 / 168 / 168.  Alternatives cost more at every row's end, but each thread
// that has one has its share of the row read again, which is shorter the more there are: with 5 at 65536 x 4096 201 / 300 / 503, at
// 16384 x 20000 157 / 154 / 203, at 8192 x 50000 194 / 168 / 177, at 4096 x 131072 258 / 210 / 194.  Few rows take more threads each.
static unsigned score_threads(const ScoreParams& p, size_t element) {
  const unsigned pieces = row_pieces(p, element);
  unsigned threads = p.top == 0 ? (pieces < 8192 ? 64 : 128) : pieces < 1024 ? 64 : pieces < 8192 ? 128 : 256;
  while (threads < 256 && (unsigned long long)p.n * threads < 1024ull * plan_sm_count() && pieces >= threads * 2) threads *= 2;
  return threads;
}

// How many blocks of 256 threads share a row: as many (a power of two) as give four blocks to an SM, with a piece at least for
// each of their threads.
static unsigned score_parts(const ScoreParams& p, size_t element, unsigned most) {
  const unsigned pieces = row_pieces(p, element);
  unsigned parts = 1;
  while (parts < most && (unsigned long long)p.n * parts * 2 <= 4ull * plan_sm_count() && pieces / (parts * 2) >= 256) parts *= 2;
  return parts;
}

template <typename T, bool TOP>
static int launch_score(const ScoreParams& p, cudaStream_t st) {
  const unsigned pieces = row_pieces(p, sizeof(T));
  constexpr int kMost = TOP && sizeof(T) == 2 ? kWarpPieces / 2 : kWarpPieces;
  if (pieces <= kMost) {
    const unsigned grid = (p.n + kWarpRows - 1) / kWarpRows, block = 32 * kWarpRows;
    if (pieces <= 32) score_warp_kernel<T, 1, TOP><<<grid, block, 0, st>>>(p);
    else if (pieces <= 64) score_warp_kernel<T, 2, TOP><<<grid, block, 0, st>>>(p);
    else if (pieces <= 128) score_warp_kernel<T, 4, TOP><<<grid, block, 0, st>>>(p);
    else if constexpr (kMost > 128) score_warp_kernel<T, 8, TOP><<<grid, block, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
  } else {
    const unsigned threads = score_threads(p, sizeof(T));
    const unsigned parts = threads == 256 ? score_parts(p, sizeof(T), kMaxCluster) : 1;
    if ((unsigned long long)p.n * parts > INT32_MAX) return BLSTM_E_TOO_LARGE;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {parts, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = p.n * parts;
    cfg.blockDim = threads;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    if (threads == 64) BLSTM_CUDA_OK(cudaLaunchKernelEx(&cfg, score_kernel<T, TOP, 64>, p));
    else if (threads == 128) BLSTM_CUDA_OK(cudaLaunchKernelEx(&cfg, score_kernel<T, TOP, 128>, p));
    else BLSTM_CUDA_OK(cudaLaunchKernelEx(&cfg, score_kernel<T, TOP, 256>, p));
  }
  count_launch();
  return BLSTM_OK;
}

}  // namespace blstm

using namespace blstm;

extern "C" {

int blstm_token_log_probs(const blstm_score_desc* d, const void* logits, const void* tokens, float* log_probs, float* entropy,
                          float* top_log_probs, int64_t* top_tokens, float* stats, void* stream) {
  if (int rc = check_score(d, logits, tokens)) return rc;
  if (d->n0 == 0 || d->n1 == 0) return BLSTM_OK;
  if (!log_probs || !entropy || (d->top && (!top_log_probs || !top_tokens)) || !aligned(4, log_probs, entropy, top_log_probs, stats) || !aligned(8, top_tokens))
    return BLSTM_E_INVALID_ARG;
  ScoreParams p = score_params(*d, logits, tokens);
  p.log_probs = log_probs; p.entropy = entropy; p.stats = stats;
  p.top_log_probs = top_log_probs; p.top_tokens = reinterpret_cast<long long*>(top_tokens);
  p.mailbox = current_mailbox();
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    return d->top ? launch_score<T, true>(p, (cudaStream_t)stream) : launch_score<T, false>(p, (cudaStream_t)stream);
  });
}

int blstm_token_log_probs_grad(const blstm_score_desc* d, const void* logits, const void* tokens, const float* stats, const int64_t* top_tokens,
                               const float* g_log_probs, const int64_t g_log_probs_stride[2], const float* g_entropy,
                               const int64_t g_entropy_stride[2], const float* g_top, void* dlogits, const int64_t dlogits_stride[2],
                               void* stream) {
  if (int rc = check_score(d, logits, tokens)) return rc;
  if (d->n0 == 0 || d->n1 == 0) return BLSTM_OK;
  if (!aligned(4, stats, g_log_probs, g_entropy, g_top) || !aligned(8, top_tokens) || !stats || !dlogits || !dlogits_stride || (g_log_probs && !g_log_probs_stride) || (g_entropy && !g_entropy_stride) || (g_top && (!top_tokens || d->top == 0)) ||
      ((reinterpret_cast<uintptr_t>(dlogits) - reinterpret_cast<uintptr_t>(logits)) & 15u) ||
      (d->n0 > 1 && ((dlogits_stride[0] - d->logits_stride[0]) * dtype_bytes(d->dtype) & 15)) ||
      (d->n1 > 1 && ((dlogits_stride[1] - d->logits_stride[1]) * dtype_bytes(d->dtype) & 15)))
    return BLSTM_E_INVALID_ARG;
  ScoreParams p = score_params(*d, logits, tokens);
  p.dlogits = dlogits;
  p.drows = row_map(d->n0, d->n1, dlogits_stride);
  p.stats = const_cast<float*>(stats);
  p.top_tokens = reinterpret_cast<long long*>(const_cast<int64_t*>(top_tokens));
  p.g_lp = g_log_probs; p.g_h = g_entropy; p.g_top = g_top;
  if (g_log_probs) p.g_lp_map = row_map(d->n0, d->n1, g_log_probs_stride);
  if (g_entropy) p.g_h_map = row_map(d->n0, d->n1, g_entropy_stride);
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    const unsigned grid = (p.n + kWarpRows - 1) / kWarpRows, block = 32 * kWarpRows, pieces = row_pieces(p, sizeof(T));
    if (pieces <= 32) score_grad_warp_kernel<T, 1><<<grid, block, 0, st>>>(p);
    else if (pieces <= 64) score_grad_warp_kernel<T, 2><<<grid, block, 0, st>>>(p);
    else if (pieces <= 128) score_grad_warp_kernel<T, 4><<<grid, block, 0, st>>>(p);
    else if (sizeof(T) == 4 && pieces <= kWarpPieces) score_grad_warp_kernel<float, 8><<<grid, block, 0, st>>>(p);
    else {
      // small blocks for short rows, so that every thread has a few pieces
      const unsigned threads = pieces <= 64 * kGradPieces ? 64 : pieces <= 128 * kGradPieces ? 128 : 256;
      p.parts = std::max(score_parts(p, sizeof(T), 1 << 16), (pieces + threads * kGradPieces - 1) / (threads * kGradPieces));
      if ((unsigned long long)p.n * p.parts > INT32_MAX) return BLSTM_E_TOO_LARGE;
      if (threads == 64) score_grad_kernel<T, 64><<<p.n * p.parts, threads, 0, st>>>(p);
      else if (threads == 128) score_grad_kernel<T, 128><<<p.n * p.parts, threads, 0, st>>>(p);
      else score_grad_kernel<T, 256><<<p.n * p.parts, threads, 0, st>>>(p);
    }
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}

}  // extern "C"
