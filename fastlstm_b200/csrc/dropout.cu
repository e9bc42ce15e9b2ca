// Dropout whose mask is a function of (seed, offset, index) and is never stored: backward draws it again.
//
//   word_m = Philox4x32-10(key = seed, counter = (m / 4, offset))[m % 4]        y = word_m >= p 2^32 ? x / (1 - p) : 0
//
// Philox is Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3" (2011).  m counts the elements in
// row-major order whatever the strides and the type, and only those of one step where the steps share a mask.
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
  unsigned steps;                // that share a mask
  long long in_step, out_step;
  unsigned threshold;
  float scale;
};

__device__ __forceinline__ uint4 philox(unsigned long long block, unsigned long long offset, unsigned long long seed) {
  unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
    c1 = (unsigned)b;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// A thread draws one block of four words and walks the steps that share it.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams p) {
  const long long block = (long long)blockIdx.x * blockDim.x + threadIdx.x, m0 = block * 4;
  if (m0 >= p.count) return;
  const uint4 w = philox(block, p.offset, p.seed_at ? *p.seed_at : p.seed);
  const unsigned word[4] = {w.x, w.y, w.z, w.w};
  unsigned r = (unsigned)(m0 / p.cols);
  long long c = m0 - r * p.cols;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (m0 + j >= p.count) break;
    const T* x = static_cast<const T*>(p.x) + p.in(r) + c;
    T* y = static_cast<T*>(p.y) + p.out(r) + c;
    const bool keep = word[j] >= p.threshold;
    for (unsigned s = 0; s < p.steps; ++s)
      y[s * p.out_step] = Elem<T>::from_f(keep ? Elem<T>::to_f(x[s * p.in_step]) * p.scale : 0.f);
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
  const long long grid = (p.count + 1023) / 1024;
  if (grid > INT32_MAX) return BLSTM_E_TOO_LARGE;
  return with_type(d->dtype, [&](auto t) -> int {
    dropout_kernel<decltype(t)><<<(unsigned)grid, 256, 0, st>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}
