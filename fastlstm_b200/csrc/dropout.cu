// Dropout whose mask is a function of (seed, offset, index) and is never stored: backward draws it again.
//
//   word_m = Philox4x32-10(key = seed, counter = (m / 4, offset))[m % 4]        y = word_m >= p 2^32 ? x / (1 - p) : 0
//
// Philox is Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3" (2011).  m counts the elements in
// row-major order whatever the strides and the type, and only those of one step where the steps share a mask.
#include <algorithm>

#include "language.cuh"

namespace blstm {

struct DropoutParams {
  const void* x;
  void* y;
  const long long* seed_at;      // the seed in device memory, or null: `seed`
  unsigned long long seed, offset;
  long long count;               // masked elements (of one step where steps share the mask)
  long long cols;
  RowMap in, out;                // rows of `cols` elements
  unsigned steps, each;          // that share a mask, and how many of them a block walks
  long long in_step, out_step;
  unsigned threshold;
  float scale;
};

// The words of N elements from element m0, a multiple of 4.  Blocks go through the rounds side by side, with one schedule of
// keys; `high`, the upper half of the block's number, is the same for all.
template <int N>
__device__ __forceinline__ void draw(unsigned (&w)[N], unsigned block, unsigned high, unsigned long long offset, unsigned long long seed) {
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int b = 0; b < N; b += 4) {
    w[b] = block + b / 4;
    w[b + 1] = high;
    w[b + 2] = (unsigned)offset;
    w[b + 3] = (unsigned)(offset >> 32);
  }
#pragma unroll
  for (int r = 0; r < 10; ++r) {
#pragma unroll
    for (int b = 0; b < N; b += 4) {
      const unsigned long long x = (unsigned long long)w[b] * 0xD2511F53u, y = (unsigned long long)w[b + 2] * 0xCD9E8D57u;
      w[b] = (unsigned)(y >> 32) ^ w[b + 1] ^ k0;
      w[b + 1] = (unsigned)y;
      w[b + 2] = (unsigned)(x >> 32) ^ w[b + 3] ^ k1;
      w[b + 3] = (unsigned)x;
    }
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> masked(const Pack<T, N>& x, const unsigned (&w)[N], unsigned threshold, float scale) {
  Pack<T, N> y;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float v = Elem<T>::to_f(x.v[k]) * scale;
    y.v[k] = Elem<T>::from_f(w[k] >= threshold ? v : 0.f);
  }
  return y;
}

__device__ __forceinline__ unsigned long long seed_of(const DropoutParams& p) { return p.seed_at ? *p.seed_at : p.seed; }

// Every element its own word, 16-byte pieces, kPieces a thread.  ROWS: rows of x have strides of their own.
constexpr int kPieces = 2;

template <typename T, bool ROWS>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int N = 16 / sizeof(T);
  using V = Pack<T, N>;
  const unsigned long long seed = seed_of(p);
  const long long pieces = (p.count + N - 1) / N, begin = (long long)blockIdx.x * (256 * kPieces);
  const unsigned long long blocks = (unsigned long long)begin * (N / 4);     // (a whole number of tiles: no carry inside of one)
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  V v[kPieces];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const long long q = begin + u * 256 + threadIdx.x, m = q * N;
    if (m + N > p.count) continue;
    long long at = m;
    if constexpr (ROWS) {
      const unsigned per_row = (unsigned)(p.cols / N);
      const unsigned r = pieces <= 0xffffffffll ? (unsigned)q / per_row : (unsigned)(q / per_row);
      at = p.in(r) + (q - (long long)r * per_row) * N;
    }
    v[u] = *reinterpret_cast<const V*>(x + at);
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const long long m = (begin + u * 256 + threadIdx.x) * N;
    if (m >= p.count) continue;
    unsigned w[N];
    draw<N>(w, (unsigned)blocks + (u * 256 + threadIdx.x) * (N / 4), (unsigned)(blocks >> 32), p.offset, seed);
    if (m + N <= p.count) *reinterpret_cast<V*>(y + m) = masked<T, N>(v[u], w, p.threshold, p.scale);
    else                                       // (not with ROWS, whose rows are whole pieces)
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (m + k < p.count) y[m + k] = Elem<T>::from_f(w[k] >= p.threshold ? Elem<T>::to_f(x[m + k]) * p.scale : 0.f);
  }
}

// Steps that share a mask: a thread draws the words of one piece and walks a part of the steps (blockIdx.y).
constexpr int kSteps = 4;            // on their way at a time

template <typename T>
__global__ void __launch_bounds__(256) dropout_shared_kernel(const __grid_constant__ DropoutParams p) {
  constexpr int N = 16 / sizeof(T);
  using V = Pack<T, N>;
  const long long q = (long long)blockIdx.x * 256 + threadIdx.x, m = q * N;
  if (m >= p.count) return;
  unsigned w[N];
  draw<N>(w, (unsigned)(m / 4), (unsigned)((unsigned long long)m >> 34), p.offset, seed_of(p));
  const unsigned r = (unsigned)(m / p.cols);
  const long long c = m - r * p.cols;
  const unsigned begin = blockIdx.y * p.each, end = min(p.steps, begin + p.each);
  const T* x = static_cast<const T*>(p.x) + p.in(r) + c + begin * p.in_step;
  T* y = static_cast<T*>(p.y) + p.out(r) + c + begin * p.out_step;
  unsigned s = begin;
  for (; s + kSteps <= end; s += kSteps) {
    V v[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) v[u] = *reinterpret_cast<const V*>(x + u * p.in_step);
#pragma unroll
    for (int u = 0; u < kSteps; ++u) *reinterpret_cast<V*>(y + u * p.out_step) = masked<T, N>(v[u], w, p.threshold, p.scale);
    x += kSteps * p.in_step;
    y += kSteps * p.out_step;
  }
  for (; s < end; ++s) {
    *reinterpret_cast<V*>(y) = masked<T, N>(*reinterpret_cast<const V*>(x), w, p.threshold, p.scale);
    x += p.in_step;
    y += p.out_step;
  }
}

// Rows that are no whole pieces, or not on 16-byte boundaries: four elements a thread, one by one.
template <typename T>
__global__ void __launch_bounds__(256) dropout_elements_kernel(const __grid_constant__ DropoutParams p) {
  const long long m0 = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 4;
  if (m0 >= p.count) return;
  unsigned w[4];
  draw<4>(w, (unsigned)(m0 / 4), (unsigned)((unsigned long long)m0 >> 34), p.offset, seed_of(p));
  unsigned r = (unsigned)(m0 / p.cols);
  long long c = m0 - r * p.cols;
  const unsigned begin = blockIdx.y * p.each, end = min(p.steps, begin + p.each);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (m0 + j >= p.count) break;
    const T* x = static_cast<const T*>(p.x) + p.in(r) + c;
    T* y = static_cast<T*>(p.y) + p.out(r) + c;
    const bool keep = w[j] >= p.threshold;
#pragma unroll 4
    for (unsigned s = begin; s < end; ++s) y[s * p.out_step] = Elem<T>::from_f(keep ? Elem<T>::to_f(x[s * p.in_step]) * p.scale : 0.f);
    if (++c == p.cols) { c = 0; ++r; }
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
  p.seed = d->seed; p.offset = d->offset;
  p.cols = d->cols;
  p.threshold = (unsigned)bound;
  p.scale = (float)(1.0 / (1.0 - d->p));
  p.steps = 1;
  const long long n1 = d->n1, C = d->cols;
  if (d->shared < 0) {
    p.count = (long long)d->n0 * n1 * C;
    p.in = row_map(n1, d->stride);
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
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | (dense ? 0 : strides * e);
  const bool pieces = (bits & 15u) == 0;
  const int per_thread = !pieces ? 4 : 16 / e * (d->shared < 0 ? kPieces : 1);
  const long long blocks = (p.count + 256ll * per_thread - 1) / (256ll * per_thread);
  if (blocks > INT32_MAX) return BLSTM_E_TOO_LARGE;
  // the steps in as many parts as give eight blocks to an SM, eight steps each at least: the words are drawn for each part
  const long long parts = std::max(1ll, std::min<long long>({8ll * plan_sm_count() / blocks, p.steps / 8, 65535}));
  p.each = (unsigned)((p.steps + parts - 1) / parts);
  const dim3 grid((unsigned)blocks, (p.steps + p.each - 1) / p.each);
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (!pieces) dropout_elements_kernel<T><<<grid, 256, 0, st>>>(p);
    else if (d->shared >= 0) dropout_shared_kernel<T><<<grid, 256, 0, st>>>(p);
    else if (dense) dropout_kernel<T, false><<<grid, 256, 0, st>>>(p);
    else dropout_kernel<T, true><<<grid, 256, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}
