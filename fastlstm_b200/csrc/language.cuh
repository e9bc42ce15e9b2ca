// What the operators around a language model share: rows of strided tensors, tokens and what is wrong with them, elements
// moved several at a time.
#pragma once

#include "common.cuh"

namespace blstm {

// Row r of a tensor [n0, n1, ...]: r = i0 * n1 + i1, strides in elements.
struct RowMap {
  long long s0, s1;
  unsigned n1;
  __device__ __forceinline__ long long operator()(unsigned r) const {
    if (r < n1) return r * s1;
    const unsigned i0 = r / n1;
    return i0 * s0 + (r - i0 * n1) * s1;
  }
};
// (rows that one stride describes are one dimension, without a division)
inline RowMap row_map(int64_t n0, int64_t n1, const int64_t stride[2]) {
  if (stride[0] == n1 * stride[1]) n1 *= n0;
  return {(long long)stride[0], (long long)stride[1], (unsigned)n1};
}

struct Tokens {
  const void* p;
  RowMap map;
  bool wide;                 // 64-bit, else 32
  __device__ __forceinline__ long long operator()(unsigned r) const {
    const long long i = map(r);
    return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
  }
};

// The mailbox that the calling thread has set (blstm_set_mailbox), or null.
int* current_mailbox();

// A token outside of the vocabulary: one report is kept, position and token in one store, the status word last.  (A mailbox of
// ints need not lie on 8 bytes: there, position and token of two reports at a time may mix.)
static __device__ __noinline__ void report_token(int* mailbox, unsigned position, long long token) {
  if (!mailbox) return;
  volatile int* m = mailbox;
  const int shown = token > INT32_MAX ? INT32_MAX : token < INT32_MIN ? INT32_MIN : (int)token;
  if ((reinterpret_cast<uintptr_t>(mailbox) & 7) == 0) {
    *reinterpret_cast<volatile unsigned long long*>(m + 2) = (unsigned long long)(unsigned)shown << 32 | position;
  } else {
    m[2] = (int)position;
    m[3] = shown;
  }
  __threadfence_system();
  m[1] = BLSTM_E_TOKEN;
}

// VEC elements of T on their natural boundary, as floats.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// The elements of a 16-byte piece as floats, and back.
template <typename T> constexpr int kPer = 16 / (int)sizeof(T);        // elements of a 16-byte piece

__device__ __forceinline__ void unpack(const uint4& v, float* z, float) {
  z[0] = __uint_as_float(v.x); z[1] = __uint_as_float(v.y); z[2] = __uint_as_float(v.z); z[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float* z, __nv_bfloat16) {
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { z[2 * i] = __uint_as_float(w[i] << 16); z[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void unpack(const uint4& v, float* z, __half) {
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    z[2 * i] = f.x; z[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack(const float* z, float) { return make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3])); }
__device__ __forceinline__ unsigned two(float a, float b, __nv_bfloat16) { const __nv_bfloat162 v = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const unsigned*>(&v); }
__device__ __forceinline__ unsigned two(float a, float b, __half) { const __half2 v = __floats2half2_rn(a, b); return *reinterpret_cast<const unsigned*>(&v); }
template <typename T>
__device__ __forceinline__ uint4 pack(const float* z, T t) { return make_uint4(two(z[0], z[1], t), two(z[2], z[3], t), two(z[4], z[5], t), two(z[6], z[7], t)); }

// Whether all addresses are multiples of `bytes`, a power of two.
template <typename... P>
bool aligned(size_t bytes, const P*... p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & (bytes - 1)) == 0; }

inline bool valid_dtype(int dtype) { return dtype == BLSTM_F32 || dtype == BLSTM_F16 || dtype == BLSTM_BF16; }
inline int dtype_bytes(int dtype) { return dtype == BLSTM_F32 ? 4 : 2; }
inline bool valid_rows(int64_t n0, int64_t n1) { return n0 >= 0 && n1 >= 0 && (n0 == 0 || n1 <= INT32_MAX / n0); }

// The widest piece, of 16, 4 and the element's own bytes, that addresses and lengths (in bytes) are multiples of.
inline int piece_bytes(uintptr_t bits, int element) { return (bits & 15u) == 0 ? 16 : (bits & 3u) == 0 ? 4 : element; }

// f(T{}) with the element type of a dtype code.
template <typename F>
int with_type(int dtype, F&& f) {
  if (dtype == BLSTM_F32) return f(float{});
  if (dtype == BLSTM_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

}  // namespace blstm
