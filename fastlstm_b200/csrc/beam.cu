// A step of beam search: the best continuations of every sentence's hypotheses, and the reordering of what belongs to them.
//
//   total[k,v] = score_k + z_kv - log sum_j exp z_kj       (an ended hypothesis: score_k for the end token, -inf for all others)
//   rank = total / length^penalty                          the `width` largest, equal ones by (k, v)
//
// Two launches.  The first reads every hypothesis' logits once, in as many parts as there are SMs for, and keeps of each part the softmax's
// statistics and the largest logits of its threads in groups.  The second has a block for every sentence: the `width`-th largest of the
// groups' totals, taken over all hypotheses, is a lower bound of the `width`-th largest total, and only the few groups that reach it are read
// again.  Bound by memory; few sentences are two chains of latencies.  Totals are compared in 64 bits, so that what decides between two
// hypotheses is the sum's error alone: 2^-24 a term, 2^-22 an exponential, which average out to some 1e-7.  (A choice: exponentials of the fast
// unit, at 67 % of its rate already, in sums of 32 bits.  Scores are 32-bit numbers: 2.3e-8 off with all in 64 bits, 2.7e-8 to 3.6e-8 so.)
#include <algorithm>

#include "score.cuh"

namespace blstm {

struct BeamParams {
  const void* logits;
  RowMap rows;
  const float* scores;
  const uint8_t* finished;       // or null
  const long long* lengths;      // or null
  unsigned batch, beams, vocab, width, parts, log_parts;       // parts of a row, a power of two
  long long end;
  double penalty;
  float2* stats;                 // [batch*beams*parts]: largest logit, sum of exp(z - it)
  float* largest;                // [batch*beams*parts][groups]
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

// NT threads have a part of a row: a warp, or a block.  Their pieces are neighbours in turns of NT; groups of NT / groups threads.
constexpr int kBlock = 256, kMostGroups = 64, kAhead = 4;
template <int NT> constexpr int kGroups = NT < kMostGroups ? NT : kMostGroups;

template <typename T, int NT>
__global__ void __launch_bounds__(kBlock) beam_rows_kernel(const __grid_constant__ BeamParams p) {
  __shared__ Sum s_part[kBlock / 32];
  constexpr int kEach = kBlock / NT, kLanes = NT / kGroups<NT>;
  const unsigned seg = blockIdx.x * kEach + threadIdx.x / NT, tid = threadIdx.x % NT, lane = tid & 31;
  const unsigned r = seg / p.parts, part = seg - r * p.parts;
  let_begin();
  if (r >= p.batch * p.beams || !goes_on(p, r)) return;          // (the same for all NT threads)
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  const Span<T> span(row, p.vocab, part, p.parts);
  const uint4* body = span.body();
  auto fetch = [&](unsigned i, uint4 (&v)[kAhead]) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = i + u * NT < span.end ? load_once(body + i + u * NT) : minus_infinity(T{});
  };
  uint4 next[kAhead];
  fetch(span.begin + tid, next);
  Sum a{-INFINITY, 0.f};
  if (tid < span.edges()) {
    const float z[2] = {ld_f(row + span.edge(tid)), -INFINITY};
    take(a, z);
  }
  for (unsigned i = span.begin + tid; i < span.end; i += kAhead * NT) {
    float z[kAhead * kPer<T>];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) unpack(next[u], z + u * kPer<T>, T{});
    fetch(i + kAhead * NT, next);
    take(a, z);
  }
  float most = a.m;
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) most = max_nan(most, __shfl_xor_sync(~0u, most, o));
  if (tid % kLanes == 0) p.largest[(size_t)seg * kGroups<NT> + tid / kLanes] = most;
  a.join(32);
  if constexpr (NT > 32) {
    if (lane == 0) s_part[tid / 32] = a;
    __syncthreads();
    a = s_part[lane % (NT / 32)];
    a.join(NT / 32);
  }
  if (tid == 0) p.stats[seg] = make_float2(a.m, a.s);
}

// Larger ranks have larger keys, NaN the largest; no key is 0.
__device__ __forceinline__ unsigned long long rank_key(double v) {
  if (v != v) return ~0ull;
  const long long b = __double_as_longlong(v + 0.0);
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 1ull << 63;
}
__device__ __forceinline__ unsigned rank_key(float v) {
  if (v != v) return ~0u;
  const unsigned b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr unsigned long long kImpossible = 0x000fffffffffffffull;      // the key of -inf
constexpr unsigned kImpossible32 = 0x007fffffu;

constexpr int kMergeThreads = 1024, kCand = 1024, kWindow = 2048, kTop = 64;

// What is among the best is decided in 64 bits; which groups are looked at, and which of their logits, in 32, with a margin for what those are
// off.  The block's code runs once, and fetching it takes most of its time (some 240 clocks for eight instructions): so many threads, few
// instructions, and loops that stay loops.
struct MergeShared {
  double base[BLSTM_MAX_BEAMS], weight[BLSTM_MAX_BEAMS];         // total = base + (z - high), rank = total weight
  float base32[BLSTM_MAX_BEAMS], weight32[BLSTM_MAX_BEAMS], high[BLSTM_MAX_BEAMS];
  int kind[BLSTM_MAX_BEAMS];                   // 0 goes on, 1 has ended, 2 is dead
  alignas(16) unsigned top[kTop];
  unsigned from;
  unsigned long long bound, place;
  unsigned long long keys[kCand], places[kCand];         // candidates: ranks, and (hypothesis, token); what comes first has the larger key, or
  float z[kCand];                                        // the smaller place
  unsigned owner[kWindow], owners, count;

  // A hypothesis whose continuations all come first (NaN, or +inf and, where a logit is -inf, NaN): every token of it counts.
  __device__ __forceinline__ bool first(unsigned k) const { return !(base32[k] < INFINITY); }
  __device__ __forceinline__ double total(unsigned k, float at) const { return base[k] == -INFINITY ? -INFINITY : base[k] + ((double)at - (double)high[k]); }
  // The rank in 32 bits, less or more (side -1, 1) than what it may be off; one that is finite stays it.  (Where nothing but -inf was found
  // there may be no token at all: as little as -inf, and where all tokens count as much as any.)
  __device__ __forceinline__ float rank32(unsigned k, float at, float side) const {
    const float d = at - high[k], off = 2e-6f * (fabsf(base32[k]) + fabsf(d));
    if (at == -INFINITY) return side > 0.f && first(k) ? -kLowest : at;
    return fminf(max_nan(max_nan(base32[k] + d + side * off, kLowest) * weight32[k], kLowest), -kLowest);
  }
  // A continuation that may be among the best.
  __device__ __noinline__ void offer(unsigned k, unsigned token, float at) {
    const unsigned long long rank = rank_key((kind[k] == 1 ? base[k] : total(k, at)) * weight[k]), at_place = (unsigned long long)k << 32 | token;
    if (rank <= kImpossible || rank < bound || (rank == bound && at_place > place)) return;
    const unsigned i = atomicAdd(&count, 1u);
    if (i >= kCand) return;
    keys[i] = rank;
    places[i] = at_place;
    z[i] = at;
  }
};

template <typename T, int NT>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ BeamParams p) {
  __shared__ MergeShared s;
  constexpr int kLanes = NT / kGroups<NT>;
  const unsigned b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r0 = b * p.beams, segs = p.beams * p.parts;
  // eight lanes have a hypothesis
  static_assert(kMergeThreads >= 8 * BLSTM_MAX_BEAMS && kMergeThreads == 16 * kTop, "");
  const unsigned mine = tid / 8;
  float score = -INFINITY;
  bool ended = false;
  if (mine < p.beams) {
    score = p.scores[r0 + mine];
    ended = p.finished && p.finished[r0 + mine];
  }
  const bool live = !ended && score != -INFINITY;
  if (mine < p.beams && tid % 8 == 0) {
    s.kind[mine] = ended ? 1 : live ? 0 : 2;
    // (from 1 to 2^24, so that a weight of 32 bits is between 2^-96 and 1 and products with it have all of their bits)
    const double weight = p.penalty != 0.0 ? 1.0 / pow((double)max(min(p.lengths[r0 + mine], (1ll << 24) - !ended) + !ended, 1ll), p.penalty) : 1.0;
    s.weight[mine] = weight;
    s.weight32[mine] = (float)weight;
  }
  if (tid < kTop) s.top[tid] = 0;
  if (tid == 0) { s.bound = 0; s.place = ~0ull; s.count = 0; s.from = ~0u; }
  let_begin();
  begin_behind();                              // (what does not need the rows' results came before)
  Sum a{-INFINITY, 0.f};
  if (live)
#pragma unroll 1
    for (unsigned q = tid % 8; q < p.parts; q += 8) {
      const float2 st = p.stats[(size_t)(r0 + mine) * p.parts + q];
      Sum o{st.x, st.y};
      const float m = max_nan(a.m, o.m), to = max_nan(m, kLowest);
      a.rescale(to);
      o.rescale(to);
      a = Sum{m, a.s + o.s};
    }
  a.join(8);
  if (mine < p.beams && tid % 8 == 0) {
    const double base = !live ? (double)score : a.s == 0.f && score < INFINITY ? -INFINITY : (double)score - log((double)a.s);      // (a row of nothing but -inf)
    s.base[mine] = base;
    s.base32[mine] = base == -INFINITY ? -INFINITY : max_nan((float)base, kLowest);                // (-inf alone stands for none)
    s.high[mine] = live ? a.m : 0.f;
  }
  __syncthreads();
  // the groups of all parts of all hypotheses by their number, without those of hypotheses that do not go on
  const float* largest = p.largest + (size_t)r0 * p.parts * kGroups<NT>;
  const unsigned all = segs * kGroups<NT>;
  auto group_key = [&](unsigned i, float side) {
    const unsigned k = i / kGroups<NT> >> p.log_parts;
    return s.kind[k] == 0 && s.base32[k] != -INFINITY ? rank_key(s.rank32(k, largest[i], side)) : 0u;
  };
  // the `width`-th largest of what they come to
  {
    unsigned most = 0;
#pragma unroll 1
    for (unsigned i = tid; i < all; i += kMergeThreads) most = max(most, group_key(i, -1.f));
    atomicMax(&s.top[tid % kTop], most);
    if (tid < p.beams && s.kind[tid] == 1) atomicMax(&s.top[tid % kTop], rank_key(s.rank32(tid, 0.f, -1.f)));
  }
  __syncthreads();
  {
    // the smallest that fewer than `width` are above (equal ones count alike): sixteen lanes have one
    const unsigned g = s.top[tid / 16];
    const uint4 v = *reinterpret_cast<const uint4*>(s.top + tid % 16 * 4);
    unsigned above = (v.x > g) + (v.y > g) + (v.z > g) + (v.w > g);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) above += __shfl_xor_sync(~0u, above, o);
    if (tid % 16 == 0 && above < p.width) atomicMin(&s.from, g);
  }
  __syncthreads();
  unsigned from = s.from;
  // what a group has of a part is looked at by warps, kRows turns of NT pieces at a time
  constexpr unsigned kRows = 32 / kLanes;
  const unsigned looks = ((p.vocab / kPer<T> >> p.log_parts) + kRows * NT) / (kRows * NT);      // (turns of a part: pieces / parts, rounded up, / NT)
  for (;;) {
    // the least rank that is looked at (-inf: all that is possible)
    const float rank = from <= kImpossible32 ? -INFINITY : __uint_as_float(from & 0x80000000u ? from & 0x7fffffffu : ~from);
    const unsigned least_key = max(from, kImpossible32 + 1);
    if (tid < p.beams && s.kind[tid] == 1) s.offer(tid, (unsigned)p.end, 0.f);
    for (unsigned w0 = 0; w0 < all; w0 += kWindow) {
      if (tid == 0) s.owners = 0;
      __syncthreads();
      const unsigned w1 = min(all, w0 + kWindow);
#pragma unroll 1
      for (unsigned i = w0 + tid; i < w1; i += kMergeThreads)
        if (group_key(i, 1.f) >= least_key) s.owner[atomicAdd(&s.owners, 1u)] = i;
      __syncthreads();
      const unsigned owners = s.owners;
#pragma unroll 1
      for (unsigned o = warp; o < owners * looks; o += kMergeThreads / 32) {
        const unsigned look = o / owners, i = s.owner[o - look * owners], seg = i / kGroups<NT>, group = i % kGroups<NT>, k = seg >> p.log_parts;
        const T* row = static_cast<const T*>(p.logits) + p.rows(r0 + k);
        const Span<T> span(row, p.vocab, seg & (p.parts - 1), p.parts);
        const unsigned piece = span.begin + (look * kRows + lane / kLanes) * NT + group * kLanes + lane % kLanes;
        const uint4 v = piece < span.end ? span.body()[piece] : minus_infinity(T{});
        // the least logit that is looked at
        const float total = rank / s.weight32[k], need = total - s.base32[k] + s.high[k];
        const float off = 4e-6f * (fabsf(total) + fabsf(s.base32[k]) + fabsf(s.high[k])) + 1e-30f, least = need - off > kLowest ? need - off : -INFINITY;
        float z[kPer<T>], m;
        unpack(v, z, T{});
        m = z[0];
#pragma unroll
        for (int e = 1; e < kPer<T>; ++e) m = max_nan(m, z[e]);
        unsigned token = span.number(piece), last = piece < span.end && (s.first(k) || !(m < least || m == -INFINITY)) ? token + kPer<T> : token;
        if (look == 0) {                       // thread `edge` of the part had one of its edges
          const unsigned edge = group * kLanes + lane;
          if (lane < kLanes && edge < span.edges()) s.offer(k, span.edge(edge), ld_f(row + span.edge(edge)));
        }
#pragma unroll 1
        for (; token < last; ++token) {        // (few, so in little code)
          const float at = ld_f(row + token);
          if (!(at < least)) s.offer(k, token, at);
        }
      }
      __syncthreads();
    }
    if (s.count <= kCand) break;
    // (many equal ones) a higher bound, the `width`-th of some of them, until they fit
    unsigned long long key = 0, at = 0;
    bool is = false;
    for (unsigned i = tid; i < kCand; i += kMergeThreads) {
      unsigned before = 0;
#pragma unroll 1
      for (unsigned j = 0; j < kCand; ++j) before += s.keys[j] > s.keys[i] || (s.keys[j] == s.keys[i] && s.places[j] < s.places[i]);
      if (before + 1 == p.width) { key = s.keys[i]; at = s.places[i]; is = true; }
    }
    __syncthreads();
    if (is) { s.bound = key; s.place = at; }
    if (tid == 0) s.count = 0;
    __syncthreads();
    const unsigned long long high = s.bound;
    // (groups that hold NaN or infinity have the largest rank that is finite)
    const double raised = __longlong_as_double((long long)(high >> 63 ? high & ~(1ull << 63) : ~high));
    from = max(from, rank_key(raised != raised ? -kLowest : fminf(fmaxf(__double2float_rd(raised), kLowest), -kLowest)));
  }
  const unsigned count = s.count;
  auto put = [&](unsigned place, unsigned k, unsigned token, double total) {
    const size_t at = (size_t)b * p.width + place;
    const bool ended = s.kind[k] == 1;
    p.out_scores[at] = (float)total;
    p.parents[at] = k;
    p.tokens[at] = token;
    if (p.out_finished) p.out_finished[at] = ended || token == p.end;
    if (p.out_lengths) p.out_lengths[at] = p.lengths[r0 + k] + !ended;
  };
  for (unsigned i0 = 0; i0 < count; i0 += kMergeThreads / 8) {         // eight lanes count what comes before a candidate
    const unsigned i = i0 + tid / 8;
    unsigned before = 0;
    if (i < count) {
      const unsigned long long key = s.keys[i], place = s.places[i];
#pragma unroll 1
      for (unsigned j = tid % 8; j < count; j += 8) before += s.keys[j] > key || (s.keys[j] == key && s.places[j] < place);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) before += __shfl_xor_sync(~0u, before, o);
    if (i < count && tid % 8 == 0 && before < p.width) {
      const unsigned k = (unsigned)(s.places[i] >> 32);
      put(before, k, (unsigned)s.places[i], s.kind[k] == 1 ? s.base[k] : s.total(k, s.z[i]));
    }
  }
  if (count >= p.width) return;
  // Too few that are possible: impossible ones follow, the first of them (no more than `count` possible ones lie between).
  if (warp == 0) {
    unsigned found = count;
    for (unsigned long long i0 = 0; found < p.width && i0 < (unsigned long long)p.beams * p.vocab; i0 += 32) {
      const unsigned long long i = i0 + lane;
      const unsigned k = (unsigned)(i / p.vocab), token = (unsigned)(i - (unsigned long long)k * p.vocab);
      bool is = k < p.beams;
      double v = -INFINITY;
      if (is && s.base[k] != -INFINITY) {
        if (s.kind[k] == 0) v = s.total(k, ld_f(static_cast<const T*>(p.logits) + p.rows(r0 + k) + token));
        else if (token == p.end) v = s.base[k];
      }
      if (is) is = rank_key(v * s.weight[k]) <= kImpossible;
      const unsigned who = __ballot_sync(~0u, is), place = found + __popc(who & ((1u << lane) - 1));
      if (is && place < p.width) put(place, k, token, v);
      found += __popc(who);
    }
  }
}

// ---------------------------------------------------------------- reordering
// Rows are moved by groups of 1 to 32 lanes, up to kRowPieces pieces a lane; longer ones in parts.  (A thread for every piece finds its row
// by divisions: 2 x 2560 rows of 301 fp32 twice and 100 x 2560 numbers 26 us, so 8, from the L2.)
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
  let_begin();
  begin_behind();                              // (a step of beam search, or whatever the stream has in front)
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
// (continuations of a sentence are counted in 32 bits)
static int check_beam(const blstm_beam_desc* d) {
  if (!d || !valid_dtype(d->dtype) || !valid_rows(d->batch, d->beams) || d->beams <= 0 || d->beams > BLSTM_MAX_BEAMS || d->width <= 0 ||
      d->width > BLSTM_MAX_TOP || d->vocab <= 0 || d->vocab >= INT32_MAX || d->beams * d->vocab > UINT32_MAX || d->width > d->beams * d->vocab || d->end_token < -1 ||
      d->end_token >= d->vocab || !(d->length_penalty >= 0 && d->length_penalty <= BLSTM_MAX_LENGTH_PENALTY) || d->batch > INT32_MAX / BLSTM_MAX_TOP)
    return BLSTM_E_INVALID_ARG;
  return BLSTM_OK;
}

// 16-byte pieces of a row: what they are at least, and at most where it does not begin on a boundary.
static unsigned beam_pieces(const blstm_beam_desc& d) { return (unsigned)((uint64_t)d.vocab * dtype_bytes(d.dtype) / 16); }

// Threads of a part, and parts of a row: warps have short rows, longer ones too where there are many; else as many parts (a power of
// two) as give kPartBlocks blocks to an SM, with kPartPieces pieces at least for each thread.  (132 x 24 x 5288 bf16 with a block and with
// a warp for each row 33 and 29 us, 256 x 4 x 2500 14.8 and 12.7, 64 x 16 x 20000 25.8 and 27.6.)
constexpr unsigned kShortPieces = 256, kManyPieces = 1024, kManyRows = 4, kPartBlocks = 16, kPartPieces = 4, kMostParts = 16;
static unsigned beam_threads(const blstm_beam_desc& d) {
  const bool many = (uint64_t)d.batch * d.beams >= (uint64_t)kManyRows * plan_sm_count();
  return beam_pieces(d) <= (many ? kManyPieces : kShortPieces) ? 32 : kBlock;
}
static unsigned beam_parts(const blstm_beam_desc& d) {
  unsigned parts = 1;
  if (beam_threads(d) == kBlock)
    while (parts < kMostParts && (uint64_t)d.batch * d.beams * parts * 2 <= (uint64_t)kPartBlocks * plan_sm_count() && beam_pieces(d) / (parts * 2) >= kPartPieces * kBlock)
      parts *= 2;
  return parts;
}
static uint64_t beam_segs(const blstm_beam_desc& d) { return (uint64_t)d.batch * d.beams * beam_parts(d); }
static size_t stats_bytes(const blstm_beam_desc& d) { return round_up(beam_segs(d) * sizeof(float2), 256); }

// A launch that may begin while the one in front of it ends (and waits for it in begin_behind).
template <typename P>
static cudaError_t launch_behind(void (*kernel)(P), unsigned grid, unsigned block, cudaStream_t st, const P& p) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int NT>
static int launch_beam(const BeamParams& p, cudaStream_t st) {
  const uint64_t segs = (uint64_t)p.batch * p.beams * p.parts, grid = (segs + kBlock / NT - 1) / (kBlock / NT);
  if (grid > INT32_MAX) return BLSTM_E_TOO_LARGE;
  beam_rows_kernel<T, NT><<<(unsigned)grid, kBlock, 0, st>>>(p);
  BLSTM_CUDA_OK(cudaGetLastError());
  BLSTM_CUDA_OK(launch_behind(beam_merge_kernel<T, NT>, p.batch, kMergeThreads, st, p));
  count_launch(2);
  return BLSTM_OK;
}

}  // namespace blstm

using namespace blstm;

extern "C" {

size_t blstm_beam_workspace(const blstm_beam_desc* d) {
  if (check_beam(d) || d->batch == 0) return 0;
  return round_up(stats_bytes(*d) + beam_segs(*d) * std::min<size_t>(beam_threads(*d), kMostGroups) * sizeof(float), 256);
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
  p.batch = (unsigned)d->batch; p.beams = (unsigned)d->beams; p.vocab = (unsigned)d->vocab; p.width = (unsigned)d->width; p.parts = beam_parts(*d);
  while (1u << p.log_parts < p.parts) ++p.log_parts;
  p.end = d->end_token;
  p.penalty = d->length_penalty;
  p.stats = static_cast<float2*>(workspace);
  p.largest = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(*d));
  p.out_scores = out_scores;
  p.parents = reinterpret_cast<long long*>(parents); p.tokens = reinterpret_cast<long long*>(tokens);
  p.out_lengths = reinterpret_cast<long long*>(out_lengths);
  p.out_finished = out_finished;
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    return beam_threads(*d) == 32 ? launch_beam<T, 32>(p, (cudaStream_t)stream) : launch_beam<T, kBlock>(p, (cudaStream_t)stream);
  });
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
    BLSTM_CUDA_OK(launch_behind(reorder_kernel, (unsigned)blocks, kReorderThreads, (cudaStream_t)stream, p));
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
    // (the kernel goes up to two parts of 32 lanes past a row's end in 32 bits)
    if (per_row > UINT32_MAX - 64 * kRowPieces || (uint64_t)s.outer > (1ull << 48) / rows / per_row) return BLSTM_E_TOO_LARGE;
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
