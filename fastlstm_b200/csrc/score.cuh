// What reads of logits share: a row in 16-byte pieces, the order of its largest logits, and how a warp, a block or a cluster finds
// them.
#pragma once

#include "language.cuh"

namespace blstm {

constexpr float kLowest = -3.402823466e38f, kFar = -10000.f;

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

// How many of n keys in shared memory come before `key`.
__device__ __forceinline__ unsigned rank_of(const unsigned long long* keys, unsigned n, unsigned long long key) {
  unsigned before = 0;
#pragma unroll 16
  for (unsigned q = 0; q < n; ++q) before += keys[q] > key;
  return before;
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

// The `top` first of a warp's logits, put(place, key) each; `mine` is the value key of the lane's largest.
constexpr int kWarpRows = 8, kWarpCand = 128;

template <typename W, typename F>
__device__ __forceinline__ void warp_top(const W& w, unsigned mine, unsigned top, unsigned long long* cand, F&& put) {
  const unsigned lane = w.lane;
  // The k-th largest of the lanes' maxima is a lower bound of the k-th largest logit: what is below it is out.
  unsigned left = mine, bound, found = 0;
  do {
    bound = __reduce_max_sync(~0u, left);
    found += __popc(__ballot_sync(~0u, left == bound));
    if (left == bound) left = 0;             // (no key is 0)
  } while (found < top);
  unsigned count = 0;
  w.each([&](float z, unsigned j, bool in) {
    const unsigned key = value_key(z), who = __ballot_sync(~0u, in && key >= bound);
    const unsigned at = count + __popc(who & ((1u << lane) - 1));
    if (in && key >= bound && at < kWarpCand) cand[at] = order_key(z, j);
    count += __popc(who);
  });
  __syncwarp();
  if (count <= kWarpCand) {
    for (unsigned i = lane; i < count; i += 32) {
      const unsigned long long key = cand[i];
      const unsigned before = rank_of(cand, count, key);
      if (before < top) put(before, key);
    }
  } else {                                   // (many equal logits) one after the other
    unsigned long long last = ~0ull;
    for (unsigned k = 0; k < top; ++k) {
      unsigned long long best = 0;
      w.each([&](float z, unsigned j, bool in) {
        const unsigned long long key = order_key(z, j);
        if (in && key < last && key > best) best = key;
      });
      for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
      if (lane == 0) put(k, best);
      last = best;
    }
  }
}

// ---------------------------------------------------------------- by a block, or a cluster of blocks
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
struct TopShared {
  alignas(16) unsigned group[kGroups];
  unsigned owner[NT];
  unsigned least[kGroups / 32];
  unsigned owners, count;
  unsigned long long bound;
  unsigned long long cand[kCand];
  unsigned long long best[BLSTM_MAX_TOP];               // of this block
};

// The `top` first of a block's logits in order, into s.best: threads' maxima bound them from below, the threads whose
// maximum reaches that bound (few more than `top`) have their logits looked at again.
template <typename T, int NT>
__device__ __forceinline__ void block_top(TopShared<NT>& s, const Span<T>& span, float thread_max, unsigned top) {
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

// The lists of a cluster's blocks, each of `top` keys in order, as one: how many keys of all come before `key`, which eight neighbouring
// lanes share, each of which finds how many of one list do.
__device__ __forceinline__ unsigned place_in_lists(const unsigned long long* all, unsigned long long key, unsigned parts, unsigned top) {
  const unsigned q = threadIdx.x % kMaxCluster;
  unsigned before = 0;
  if (q < parts)
#pragma unroll
    for (unsigned step = BLSTM_MAX_TOP; step; step >>= 1)
      if (before + step <= top && all[q * top + before + step - 1] > key) before += step;
#pragma unroll
  for (int o = 1; o < kMaxCluster; o <<= 1) before += __shfl_xor_sync(0xffu << (threadIdx.x & 24u), before, o);
  return before;
}

}  // namespace blstm
