// What reads of logits share: a row in 16-byte pieces, exponentials of distances from its maximum.
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

// 2^x to 2^-22; subnormal results are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

}  // namespace blstm
