// Dropout whose mask is a function of (seed, offset, index) and is never stored: backward draws it again.
//
//   word_m = Philox4x32-10(key = seed, counter = (m / 4, offset))[m % 4]        y = word_m >= p 2^32 ? x / (1 - p) : 0
//
// Philox is Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3" (2011).  m counts the elements in
// row-major order whatever the strides and the type, and only those of one step where the steps share a mask.
#include <algorithm>
#include <type_traits>

#include "language.cuh"

namespace blstm {

struct DropoutParams {
  const void* x;
  void* y;
  const long long* seed_at;      // the seed in device memory, or null
  unsigned long long offset;
  unsigned keys[20];             // of the rounds, where the seed is not in device memory
  long long count;               // masked elements (of one step where steps share the mask)
  long long cols;
  RowMap in, out;                // rows of `cols` elements
  unsigned steps, each;          // that share a mask, and how many of them a block walks
  long long in_step, out_step;
  unsigned threshold;
  float scale;
};

// The keys of the ten rounds: from the host, where they come with the parameters and cost nothing, or from a seed in device
// memory.
template <bool SEED_AT>
struct Keys {
  unsigned k[SEED_AT ? 20 : 1];
  __device__ __forceinline__ explicit Keys(const DropoutParams& p) {
    if constexpr (SEED_AT) {
      const unsigned long long seed = *p.seed_at;
#pragma unroll
      for (int r = 0; r < 10; ++r) {
        k[2 * r] = (unsigned)seed + r * 0x9E3779B9u;
        k[2 * r + 1] = (unsigned)(seed >> 32) + r * 0xBB67AE85u;
      }
    }
  }
  __device__ __forceinline__ unsigned operator()(const DropoutParams& p, int i) const { return SEED_AT ? k[SEED_AT ? i : 0] : p.keys[i]; }
};

// The words of N elements from element 4 block; `high`, the upper half of the block's number, is the same for all of them.
template <int N, bool SEED_AT>
__device__ __forceinline__ void draw(unsigned (&w)[N], const DropoutParams& p, const Keys<SEED_AT>& keys, unsigned block, unsigned high) {
#pragma unroll
  for (int b = 0; b < N; b += 4) {
    w[b] = block + b / 4;
    w[b + 1] = high;
    w[b + 2] = (unsigned)p.offset;
    w[b + 3] = (unsigned)(p.offset >> 32);
  }
#pragma unroll
  for (int r = 0; r < 10; ++r) {
#pragma unroll
    for (int b = 0; b < N; b += 4) {
      const unsigned long long x = (unsigned long long)w[b] * 0xD2511F53u, y = (unsigned long long)w[b + 2] * 0xCD9E8D57u;
      w[b] = (unsigned)(y >> 32) ^ w[b + 1] ^ keys(p, 2 * r);
      w[b + 1] = (unsigned)y;
      w[b + 2] = (unsigned)(x >> 32) ^ w[b + 3] ^ keys(p, 2 * r + 1);
      w[b + 3] = (unsigned)x;
    }
  }
}

// A piece with the elements dropped whose words are below the threshold, whatever they hold.
template <typename T>
__device__ __forceinline__ uint4 masked(const uint4& v, const unsigned (&w)[kPer<T>], const DropoutParams& p) {
  float z[kPer<T>];
  unpack(v, z, T{});
#pragma unroll
  for (int k = 0; k < kPer<T>; ++k) {
    const float y = z[k] * p.scale;
    z[k] = w[k] >= p.threshold ? y : 0.f;
  }
  return pack(z, T{});
}

// The same in two steps, for words that serve many pieces: bits that stay, and a piece with them.
template <typename T>
__device__ __forceinline__ uint4 stays(const unsigned (&w)[kPer<T>], unsigned threshold) {
  unsigned b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) b[i] = w[i] >= threshold ? ~0u : 0u;
    else b[i] = (w[2 * i] >= threshold ? 0xffffu : 0u) | (w[2 * i + 1] >= threshold ? 0xffff0000u : 0u);
  }
  return make_uint4(b[0], b[1], b[2], b[3]);
}
template <typename T>
__device__ __forceinline__ uint4 masked(const uint4& v, const uint4& bits, float scale) {
  float z[kPer<T>];
  unpack(v, z, T{});
#pragma unroll
  for (int k = 0; k < kPer<T>; ++k) z[k] *= scale;
  const uint4 y = pack(z, T{});
  return make_uint4(y.x & bits.x, y.y & bits.y, y.z & bits.z, y.w & bits.w);
}

// Every element its own word, 16-byte pieces, kPieces a thread.  ROWS: rows of x have strides of their own.
// A block of four words takes 20 products of 32 x 32 bits to 64, which an SM makes 32 lanes of a clock: 1.77e12 words/s.  256 x 512 x
// 512: fp32 81 us (6.6 TB/s: the copy bandwidth), bf16 55.6 us (4.8 TB/s), where the words alone take 38 us and the copy alone 41; with one
// piece a thread 61.6, with four 55.8, in a persistent grid with its loads ahead 57.5.
constexpr int kPieces = 2;

template <typename T, bool SEED_AT, bool ROWS>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int N = kPer<T>, kTile = 256 * kPieces;
  const Keys<SEED_AT> keys(p);
  const unsigned long long begin = (unsigned long long)blockIdx.x * kTile, whole = p.count / N;      // pieces
  const unsigned long long number = begin * (N / 4);        // Philox blocks: a whole number of tiles, no carry inside of one
  const T* x = static_cast<const T*>(p.x);
  uint4* y = static_cast<uint4*>(p.y) + begin;
  const uint4* from[kPieces];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const unsigned i = u * 256 + threadIdx.x;
    if constexpr (ROWS) {
      const unsigned per_row = (unsigned)(p.cols / N);
      const unsigned long long q = begin + i;
      const unsigned r = q <= 0xffffffffu ? (unsigned)q / per_row : (unsigned)(q / per_row);
      from[u] = reinterpret_cast<const uint4*>(x + p.in(r) + (long long)(q - (unsigned long long)r * per_row) * N);
    } else {
      from[u] = reinterpret_cast<const uint4*>(x) + begin + i;
    }
  }
  auto words = [&](unsigned (&w)[N], unsigned i) { draw(w, p, keys, (unsigned)number + i * (N / 4), (unsigned)(number >> 32)); };
  if (begin + kTile <= whole) {
    uint4 v[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) v[u] = *from[u];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      unsigned w[N];
      words(w, u * 256 + threadIdx.x);
      y[u * 256 + threadIdx.x] = masked<T>(v[u], w, p);
    }
    return;
  }
  for (int u = 0; u < kPieces; ++u) {
    const unsigned i = u * 256 + threadIdx.x;
    if (begin + i > whole) continue;
    unsigned w[N];
    words(w, i);
    if (begin + i < whole) y[i] = masked<T>(*from[u], w, p);
    else                                       // the elements behind the last piece (not with ROWS, whose rows are whole pieces)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const unsigned long long m = whole * N + k;
        if ((long long)m < p.count) static_cast<T*>(p.y)[m] = Elem<T>::from_f(w[k] >= p.threshold ? Elem<T>::to_f(x[m]) * p.scale : 0.f);
      }
  }
}

// Steps that share a mask: a thread draws the words of one piece and walks a part of the steps (blockIdx.y), all of which are
// on their way together.  Short parts keep the blocks that run at a time in neighbouring memory (512 x 256 x 1024 fp16:
// 8 steps 82.7 us, 16 84.5, 32 86.7, parts of 52 steps 92), and drawing the words again for every eighth step is hidden.
constexpr int kSteps = 8;

template <typename T, bool SEED_AT>
__global__ void __launch_bounds__(256) dropout_shared_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int N = kPer<T>;
  const long long q = (long long)blockIdx.x * 256 + threadIdx.x, m = q * N;
  if (m >= p.count) return;
  unsigned w[N];
  draw(w, p, Keys<SEED_AT>(p), (unsigned)(m / 4), (unsigned)((unsigned long long)m >> 34));
  const uint4 bits = stays<T>(w, p.threshold);
  const unsigned r = (unsigned)(m / p.cols);
  const long long c = m - r * p.cols;
  const unsigned begin = blockIdx.y * p.each, end = min(p.steps, begin + p.each);
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + p.in(r) + c + begin * p.in_step);
  uint4* y = reinterpret_cast<uint4*>(static_cast<T*>(p.y) + p.out(r) + c + begin * p.out_step);
  const long long in_step = p.in_step / N, out_step = p.out_step / N;
  for (unsigned s = begin; s < end; s += kSteps) {
    uint4 v[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) if (s + u < end) v[u] = x[u * in_step];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) if (s + u < end) y[u * out_step] = masked<T>(v[u], bits, p.scale);
    x += kSteps * in_step;
    y += kSteps * out_step;
  }
}

// Rows that are no whole pieces, or not on 16-byte boundaries.  Where every element has its own word a thread makes 16 bytes of y,
// which has no gaps, out of loads of L elements (512 x 256 x 643 turned: fp32 158 us, bf16 124, with stores as narrow as the loads
// 431 and 435).
template <typename T, bool SEED_AT, int L>
__global__ void __launch_bounds__(256) dropout_gather_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int N = kPer<T>;
  using V = Pack<T, L>;
  const long long q = (long long)blockIdx.x * 256 + threadIdx.x, m = q * N;
  if (m >= p.count) return;
  unsigned r;
  if (p.cols <= 0xffffffffll && m <= 0xffffffffll) r = (unsigned)m / (unsigned)p.cols;
  else r = (unsigned)(m / p.cols);
  long long c = m - r * p.cols;
  const T* x = static_cast<const T*>(p.x) + p.in(r) + c;
  alignas(16) T v[N];
  if (c + N <= p.cols) {
#pragma unroll
    for (int k = 0; k < N; k += L) *reinterpret_cast<V*>(v + k) = *reinterpret_cast<const V*>(x + k);
  } else if (p.cols >= N) {                    // the end of a row and the begin of the next one, or the end of all
    const T* next = static_cast<const T*>(p.x) + p.in(r + 1) - (p.cols - c);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = m + k < p.count ? (c + k < p.cols ? x : next)[k] : Elem<T>::from_f(0.f);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k, ++c) {
      if (c == p.cols) { c = 0; ++r; }
      v[k] = m + k < p.count ? static_cast<const T*>(p.x)[p.in(r) + c] : Elem<T>::from_f(0.f);
    }
  }
  unsigned w[N];
  draw(w, p, Keys<SEED_AT>(p), (unsigned)(m / 4), (unsigned)((unsigned long long)m >> 34));
  T* y = static_cast<T*>(p.y) + m;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = Elem<T>::from_f(w[k] >= p.threshold ? Elem<T>::to_f(v[k]) * p.scale : 0.f);
  if (m + N <= p.count && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {
    Pack<T, N> out;
#pragma unroll
    for (int k = 0; k < N; ++k) out.v[k] = v[k];
    *reinterpret_cast<Pack<T, N>*>(y) = out;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (m + k < p.count) y[k] = v[k];
  }
}

// Where steps share a mask a thread has one element of each: four threads draw the same block, for eight steps (512 x 255 x 643:
// fp32 119 us, bf16 115, with the four elements of a block in one thread 265 and 156).
template <typename T, bool SEED_AT>
__global__ void __launch_bounds__(256) dropout_column_kernel(const __grid_constant__ DropoutParams p) {
  const long long m = (long long)blockIdx.x * 256 + threadIdx.x;
  if (m >= p.count) return;
  unsigned w[4];
  draw(w, p, Keys<SEED_AT>(p), (unsigned)(m / 4), (unsigned)((unsigned long long)m >> 34));
  const unsigned word = m & 2 ? (m & 1 ? w[3] : w[2]) : (m & 1 ? w[1] : w[0]);
  const bool stays = word >= p.threshold;
  const unsigned r = (unsigned)(m / p.cols);
  const long long c = m - r * p.cols;
  const unsigned begin = blockIdx.y * p.each, end = min(p.steps, begin + p.each);
  const T* x = static_cast<const T*>(p.x) + p.in(r) + c + begin * p.in_step;
  T* y = static_cast<T*>(p.y) + p.out(r) + c + begin * p.out_step;
  for (unsigned s = begin; s < end; s += kSteps) {
    T v[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) if (s + u < end) v[u] = x[u * p.in_step];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) if (s + u < end) y[u * p.out_step] = Elem<T>::from_f(stays ? Elem<T>::to_f(v[u]) * p.scale : 0.f);
    x += kSteps * p.in_step;
    y += kSteps * p.out_step;
  }
}

}  // namespace blstm

using namespace blstm;

extern "C" int blstm_dropout(const blstm_dropout_desc* d, const void* x, const int64_t* seed, void* y, void* stream) {
  if (!d || !valid_dtype(d->dtype) || !valid_rows(d->n0, d->n1) || d->cols < 0 || d->shared < -1 || d->shared > 1 ||
      !(d->p >= 0.0 && d->p <= 1.0))
    return BLSTM_E_INVALID_ARG;
  if (d->n0 == 0 || d->n1 == 0 || d->cols == 0) return BLSTM_OK;
  if (!x || !y) return BLSTM_E_INVALID_ARG;
  const int e = dtype_bytes(d->dtype);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % e || reinterpret_cast<uintptr_t>(seed) % 8) return BLSTM_E_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const double bound = d->p * 4294967296.0 + 0.5;
  if (bound >= 4294967296.0) {                    // nothing stays
    BLSTM_CUDA_OK(cudaMemsetAsync(y, 0, (size_t)d->n0 * d->n1 * d->cols * e, st));
    return BLSTM_OK;
  }
  DropoutParams p{};
  p.x = x; p.y = y;
  p.seed_at = reinterpret_cast<const long long*>(seed);
  p.offset = d->offset;
  for (unsigned r = 0; r < 10; ++r) {
    p.keys[2 * r] = (unsigned)d->seed + r * 0x9E3779B9u;
    p.keys[2 * r + 1] = (unsigned)(d->seed >> 32) + r * 0xBB67AE85u;
  }
  p.cols = d->cols;
  p.threshold = (unsigned)bound;
  p.scale = (float)(1.0 / (1.0 - d->p));
  p.steps = 1;
  const long long n1 = d->n1, C = d->cols;
  if (d->shared < 0) {
    p.count = (long long)d->n0 * n1 * C;
    p.in = row_map(d->n0, n1, d->stride);
    p.out = {n1 * C, C, (unsigned)n1};
  } else if (d->shared == 0) {                    // the mask of [n1, cols], n0 times
    p.count = n1 * C;
    p.in = {0, d->stride[1], (unsigned)n1};
    p.out = {0, C, (unsigned)n1};
    p.steps = (unsigned)d->n0; p.in_step = d->stride[0]; p.out_step = n1 * C;
  } else {                                        // of [n0, cols], n1 times
    p.count = (long long)d->n0 * C;
    p.in = {d->stride[0], 0, 1};
    p.out = {n1 * C, 0, 1};
    p.steps = (unsigned)n1; p.in_step = d->stride[1]; p.out_step = C;
  }
  // 16-byte pieces need rows that are whole pieces on 16-byte boundaries; a tensor without gaps is one row, whose end may be ragged
  const bool dense = d->shared < 0 && (n1 == 1 || d->stride[1] == C) && (d->n0 == 1 || d->stride[0] == n1 * C);
  const uintptr_t strides = (d->n0 > 1 ? (uintptr_t)d->stride[0] : 0) | (d->n1 > 1 ? (uintptr_t)d->stride[1] : 0) | (uintptr_t)C;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | (dense ? 0 : strides * e) | (reinterpret_cast<uintptr_t>(y) & 15u ? 12u : 0);
  const bool pieces = (bits & 15u) == 0;
  const bool pairs = (bits & 3u) == 0 && e == 2;          // elements of 16 bits, two at a time
  const int per_thread = d->shared < 0 ? 16 / e * (pieces ? kPieces : 1) : pieces ? 16 / e : 1;
  const long long blocks = (p.count + 256ll * per_thread - 1) / (256ll * per_thread);
  if (blocks > INT32_MAX) return BLSTM_E_TOO_LARGE;
  p.each = std::max((unsigned)kSteps, (p.steps + 65534) / 65535);        // (a grid has 65535 parts at most)
  const dim3 grid((unsigned)blocks, (p.steps + p.each - 1) / p.each);
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto launch = [&](auto at) {
      constexpr bool A = decltype(at)::value;
      if (!pieces && d->shared >= 0) dropout_column_kernel<T, A><<<grid, 256, 0, st>>>(p);
      else if (!pieces && pairs) dropout_gather_kernel<T, A, 4 / sizeof(T)><<<grid, 256, 0, st>>>(p);
      else if (!pieces) dropout_gather_kernel<T, A, 1><<<grid, 256, 0, st>>>(p);
      else if (d->shared >= 0) dropout_shared_kernel<T, A><<<grid, 256, 0, st>>>(p);
      else if (dense) dropout_kernel<T, A, false><<<grid, 256, 0, st>>>(p);
      else dropout_kernel<T, A, true><<<grid, 256, 0, st>>>(p);
    };
    if (seed) launch(std::true_type{});
    else launch(std::false_type{});
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}
