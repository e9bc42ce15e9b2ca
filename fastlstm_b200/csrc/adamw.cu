// A step of AdamW (decoupled weight decay: Loshchilov, Hutter, 2019) over many tensors in one launch, and the norm of all of their
// gradients.
//
//   g' = g f        m' = b1 m + (1 - b1) g'      v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// f = min(1, max_norm / (|g| + 1e-6)), where |g| is the norm over all tensors.  A tensor's count of steps t lies in device memory and
// is raised by the launch itself, so a captured step can be replayed.  Bound by memory: 28 bytes an element in fp32.
//
// States in 8 bits: 256 elements share a scale of 32 bits (their largest magnitude / 448); m and u = sqrt(v) are e4m3 numbers times
// it.  A step changes v by (1 - b2) of itself at most where gradients get smaller, far less than half the distance of two e4m3 numbers:
// rounded to the nearest it would never fall (simulated with b2 = 0.999, gradients that fall by up to two decades over 4000 steps: the root
// 6 times too large on average).  So both are cut off or rounded up by chance, the mean is what it should be, and the root stays
// within 2 % on average.  The chance is a function of seed, step, tensor and element: a run repeats bit by bit.  u is never rounded to
// 0, which would divide by it.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "language.cuh"

namespace blstm {

constexpr int kAdamThreads = 256, kTurn = 8 * kAdamThreads;       // elements of a block's turn: 8 a thread, 256 (a scale) a warp
constexpr int kChunk = 4 * kTurn;

struct AdamItem {
  void* param;
  const void* grad;
  void *m, *v;                   // fp32, or e4m3
  float *m_scale, *v_scale, *master;
  long long* step;
  long long n;
  unsigned first, number;        // its first chunk; for the words
};
template <int CAP>
struct AdamParams {
  AdamItem item[CAP];
  unsigned items, chunks;
  unsigned long long wide[(CAP + 63) / 64];            // items whose addresses are multiples of 16
  unsigned keys[20];
  float lr, beta1, beta2, one_less1, one_less2, eps, decay, one;       // one: 1 (see AdamStep)
  double log_beta1, log_beta2;
  const float *lr_at, *factor;
  unsigned* ticket;
};

// Eight elements as they lie in memory: in 16-byte pieces where all eight are there and on a boundary (WHOLE, or as `wide` and `left` say), else the
// first `left` of them one by one, zeros behind.
template <typename T>
struct Raw {
  static constexpr int N = sizeof(T) / 2;              // 16-byte pieces
  uint4 v[N];
  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* p, long long left, bool wide) {
    if (WHOLE || (wide && left >= 8)) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = reinterpret_cast<const uint4*>(p)[k];
    } else {
      float z[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k] = k < left ? ld_f(p + k) : 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = pack(z + k * kPer<T>, T{});
    }
  }
  __device__ __forceinline__ void get(float (&z)[8]) const {
#pragma unroll
    for (int k = 0; k < N; ++k) unpack(v[k], z + k * kPer<T>, T{});
  }
};
template <bool WHOLE, typename T>
__device__ __forceinline__ void store8(T* p, long long left, bool wide, const float (&z)[8]) {
  if (WHOLE || (wide && left >= 8)) {
#pragma unroll
    for (int k = 0; k < 8; k += kPer<T>) *reinterpret_cast<uint4*>(p + k) = pack(z + k, T{});
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) p[k] = Elem<T>::from_f(z[k]);
  }
}
template <bool WHOLE>
__device__ __forceinline__ uint2 load8_bytes(const uint8_t* p, long long left, bool wide) {
  if (WHOLE || (wide && left >= 8)) return *reinterpret_cast<const uint2*>(p);
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < left) w[k / 4] |= (unsigned)p[k] << k % 4 * 8;
  return make_uint2(w[0], w[1]);
}
template <bool WHOLE>
__device__ __forceinline__ void store8_bytes(uint8_t* p, long long left, bool wide, uint2 v) {
  if (WHOLE || (wide && left >= 8)) {
    *reinterpret_cast<uint2*>(p) = v;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) p[k] = (uint8_t)((k < 4 ? v.x : v.y) >> k % 4 * 8);
  }
}
__device__ __forceinline__ void decode8(uint2 w, Pair (&z)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned short two = (unsigned short)((k < 2 ? w.x : w.y) >> k % 2 * 16);
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    z[k] = Pair::of(f.x, f.y);
  }
}

// A number of at most 448, times 2^-120, as an e4m3 number in bits 20 to 26, its sign where it was: what it is in a float's own bits,
// subnormal numbers too, and adding `chance` (16 bits, of 20) below it rounds up with the probability of what is cut off.  (The division that
// makes the largest 448 is off by two in the last place at most, which no chance carries to the next number.)
__device__ __forceinline__ unsigned encode(float y, unsigned chance) { return __float_as_uint(y) + (chance << 4); }
// Four of them in their order in memory.
__device__ __forceinline__ unsigned bytes_of(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x7632) >> 4, __byte_perm(c, d, 0x7632) >> 4, 0x6420);
}
__device__ __forceinline__ unsigned signs_of(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410) & 0x80808080u;
}

// The words of elements 4 block .. 4 block + 3 in step t of tensor `number`: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) with the seed
// as the key and (block, t, number) as the counter.
__device__ __forceinline__ void draw4(unsigned (&w)[4], const unsigned* keys, unsigned long long block, unsigned t, unsigned number) {
  w[0] = (unsigned)block;
  w[1] = (unsigned)(block >> 32);
  w[2] = t;
  w[3] = number;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long x = (unsigned long long)w[0] * 0xD2511F53u, y = (unsigned long long)w[2] * 0xCD9E8D57u;
    w[0] = (unsigned)(y >> 32) ^ w[1] ^ keys[2 * r];
    w[1] = (unsigned)y;
    w[2] = (unsigned)(x >> 32) ^ w[3] ^ keys[2 * r + 1];
    w[3] = (unsigned)x;
  }
}

__device__ __forceinline__ float max_abs(float m, float v) {      // NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}
// The largest of a warp's magnitudes: their bits have their order, and NaN comes last.
__device__ __forceinline__ float warp_most(float most) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(most))); }
// (Fast roots and quotients are a choice: what they are off is 2^-21 of a step's move, which is small beside the weight.  0.7 M fp32 weights with
// their states after a step: 3.9e-8 off the numbers in 64 bits, 4.7e-8 with every operation rounded for itself.)
__device__ __forceinline__ float reciprocal_fast(float x) {      // to 2^-23; of 0, or at least 2^-126
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sqrt_fast(float x) {      // to 2^-22
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two square roots by a step of Newton's iteration from v r, r the fast unit's 1 / sqrt(v) to 2^-22: the residual v - u^2 is exact in a
// fused product, so what is left is the last rounding, and 2^-44.  0 is 0; below 2^-126 (where r is held) it is no root.
__device__ __forceinline__ Pair roots(Pair v, Pair half) {
  float lo, hi, a, b;
  v.get(lo, hi);
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(lo));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(hi));
  const Pair r = Pair::of(fminf(a, 0x1p63f), fminf(b, 0x1p63f)), u = v * r;
  return fma2(fma2(u * Pair::of(-1.f, -1.f), u, v), r * half, u);
}

// What a scale and its inverse are for a largest magnitude; magnitudes below 2^-110 are 0 (the inverse would not be a number of 32 bits).
struct Scale {
  float up, down;
  __device__ __forceinline__ explicit Scale(float most)
      : up(most > 0x1p-110f ? 1.f / most * 448.f : 0.f), down(most <= 0x1p-110f ? 0.f : most * (1.f / 448.f)) {}
};

// What a step does to eight elements.
struct AdamStep {
  float factor, beta1, beta2, one_less1, one_less2, eps, decay, one, c1, c2;

  __device__ __forceinline__ void operator()(const float (&g)[8], float (&m)[8], float (&v)[8], float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = g[e] * factor;
      m[e] = fmaf(beta1, m[e], one_less1 * ge);
      v[e] = fmaf(beta2, v[e], one_less2 * (ge * ge));
      x[e] -= fmaf(decay, x[e], c1 * m[e] * reciprocal_fast(fmaf(sqrt_fast(v[e]), c2, eps)));
    }
  }

  // The same in 8 bits, by a warp with 256 elements: m8 and u8 are theirs and become the new ones, as do the scales.  Two floats an
  // instruction (it is instructions that bound this).  Moments, roots and scales are rounded operation by operation, so that they depend on
  // the formula alone: between small numbers a step of e4m3 is half of what it is taken from, and the next step's quotient goes by it.
  template <typename F>
  __device__ __forceinline__ void operator()(const float (&g)[8], uint2& m8, uint2& u8, float& m_scale, float& u_scale, float (&x)[8], F&& words) const {
    Pair m[4], v[4], u[4];
    float most_m = 0.f, most_v = 0.f;
    decode8(m8, m);
    decode8(u8, v);
    auto both = [](float a) { return Pair::of(a, a); };
    const Pair sm = both(m_scale), su = both(u_scale), f = both(factor), b1 = both(beta1), b2 = both(beta2), a1 = both(one_less1), a2 = both(one_less2);
    // (a sum as a product with a 1 that the compiler does not know: it makes one rounding of a product and a sum, also of those that say how
    // they round)
    const Pair same = both(one), minus = both(-1.f), rate = both(c1), fix = both(c2), e0 = both(eps), wd = both(decay);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const Pair ge = Pair::of(g[2 * k], g[2 * k + 1]) * f, old = v[k] * su;
      m[k] = fma2(b1 * (m[k] * sm), same, a1 * ge);
      v[k] = fma2(b2 * (old * old), same, a2 * (ge * ge));
      float lo, hi;
      m[k].get(lo, hi);
      most_m = max_abs(max_abs(most_m, lo), hi);
      v[k].get(lo, hi);
      most_v = max_abs(max_abs(most_v, lo), hi);
      u[k] = roots(v[k], both(0.5f));
    }
    const float largest = warp_most(most_v);
    if (largest < 0x1p-56f)                     // (above it, what has a square below 2^-126 is nothing next to the scale)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float lo, hi;
        v[k].get(lo, hi);
        u[k] = Pair::of(__fsqrt_rn(lo), __fsqrt_rn(hi));
      }
    const Scale ms(warp_most(most_m)), us(__fsqrt_rn(largest));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float p, q;
      fma2(u[k], fix, e0).get(p, q);
      const Pair move = m[k] * rate * Pair::of(reciprocal_fast(p), reciprocal_fast(q)), at = Pair::of(x[2 * k], x[2 * k + 1]);
      fma2(fma2(at, wd, move), minus, at).get(x[2 * k], x[2 * k + 1]);
    }
    const Pair up_m = both(ms.up), up_u = both(us.up), small = both(0x1p-120f);
    unsigned half_m[2], half_u[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned w[4], cm[4], cu[4], least = ~0u;
      words(h, w);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float y[2], z[2];
        (m[2 * h + k] * up_m * small).get(y[0], y[1]);
        (u[2 * h + k] * up_u * small).get(z[0], z[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int e = 2 * k + i;
          cm[e] = encode(y[i], w[e] & 0xffffu);
          cu[e] = encode(z[i], w[e] >> 16);
          least = min(least, cu[e]);
        }
      }
      if (least < 1u << 20)                     // (a root that is not 0 does not become it)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float lo, hi;
          u[2 * h + k].get(lo, hi);
          if (lo > 0.f) cu[2 * k] = max(cu[2 * k], 1u << 20);
          if (hi > 0.f) cu[2 * k + 1] = max(cu[2 * k + 1], 1u << 20);
        }
      half_m[h] = bytes_of(cm[0], cm[1], cm[2], cm[3]) & 0x7f7f7f7fu | signs_of(cm[0], cm[1], cm[2], cm[3]);
      half_u[h] = bytes_of(cu[0], cu[1], cu[2], cu[3]);
    }
    m8 = make_uint2(half_m[0], half_m[1]);
    u8 = make_uint2(half_u[0], half_u[1]);
    m_scale = ms.down;
    u_scale = us.down;
  }
};

// A chunk of an item from element `begin` on, of which `left` are there: what a turn needs is fetched while the one before it is worked on.
template <typename T, int BITS, bool MASTER, bool WHOLE>
__device__ __forceinline__ void turns(const AdamStep& step, const AdamItem& a, long long begin, long long left, bool wide, const unsigned* keys, unsigned t) {
  const unsigned tid = threadIdx.x;
  const long long i0 = begin + tid * 8;
  const T* grad = static_cast<const T*>(a.grad) + i0;
  T* param = static_cast<T*>(a.param) + i0;
  float *m32 = static_cast<float*>(a.m) + i0, *v32 = static_cast<float*>(a.v) + i0, *w32 = MASTER ? a.master + i0 : nullptr;
  uint8_t *mb = static_cast<uint8_t*>(a.m) + i0, *ub = static_cast<uint8_t*>(a.v) + i0;
  float *sm = a.m_scale + i0 / 256, *su = a.v_scale + i0 / 256;        // (of a warp)
  Raw<T> g, x;
  Raw<float> m, v, master;
  uint2 m8, u8;
  float m_scale = 0.f, u_scale = 0.f;
  auto fetch = [&](int at, long long rest) {
    g.template load<WHOLE>(grad + at, rest, wide);
    if constexpr (BITS == 32) {
      m.template load<WHOLE>(m32 + at, rest, wide);
      v.template load<WHOLE>(v32 + at, rest, wide);
    } else {
      m8 = load8_bytes<WHOLE>(mb + at, rest, wide);
      u8 = load8_bytes<WHOLE>(ub + at, rest, wide);
      if (WHOLE || rest + (tid % 32) * 8 > 0) {
        m_scale = sm[at / 256];
        u_scale = su[at / 256];
      }
    }
    if constexpr (MASTER) master.template load<WHOLE>(w32 + at, rest, wide);
    else x.template load<WHOLE>(param + at, rest, wide);
  };
  long long rest = left - tid * 8;              // from this thread's first element on
  fetch(0, rest);
  const int end = WHOLE ? kChunk : (int)min(left, (long long)kChunk);
#pragma unroll 1
  for (int at = 0; at < end; at += kTurn, rest -= kTurn) {
    float ge[8], xe[8];
    g.get(ge);
    if constexpr (MASTER) master.get(xe);
    else x.get(xe);
    if constexpr (BITS == 32) {
      float me[8], ve[8];
      m.get(me);
      v.get(ve);
      if (at + kTurn < end) fetch(at + kTurn, rest - kTurn);
      step(ge, me, ve, xe);
      store8<WHOLE>(m32 + at, rest, wide, me);
      store8<WHOLE>(v32 + at, rest, wide, ve);
    } else {
      uint2 mine = m8, roots = u8;
      float ms = m_scale, us = u_scale;
      if (at + kTurn < end) fetch(at + kTurn, rest - kTurn);
      step(ge, mine, roots, ms, us, xe, [&](int h, unsigned (&w)[4]) { draw4(w, keys, (unsigned long long)(i0 + at) / 4 + h, t, a.number); });
      store8_bytes<WHOLE>(mb + at, rest, wide, mine);
      store8_bytes<WHOLE>(ub + at, rest, wide, roots);
      if (tid % 32 == 0 && (WHOLE || rest > 0)) {
        sm[at / 256] = ms;
        su[at / 256] = us;
      }
    }
    if constexpr (MASTER) store8<WHOLE>(w32 + at, rest, wide, xe);
    store8<WHOLE>(param + at, rest, wide, xe);
  }
}

// Which chunk a block is at, and the item that it belongs to.
template <int CAP>
struct Cursor {
  unsigned chunk, k = 0;
  __device__ __forceinline__ Cursor() : chunk(blockIdx.x) {}
  __device__ __forceinline__ bool there(const AdamParams<CAP>& p) {
    if (chunk >= p.chunks) return false;
    while (k + 1 < p.items && chunk >= p.item[k + 1].first) ++k;
    return true;
  }
  __device__ __forceinline__ long long begin(const AdamParams<CAP>& p) const { return (long long)(chunk - p.item[k].first) * kChunk; }
  __device__ __forceinline__ bool wide(const AdamParams<CAP>& p) const { return p.wide[k / 64] >> k % 64 & 1; }
  __device__ __forceinline__ bool whole(const AdamParams<CAP>& p) const { return wide(p) && p.item[k].n - begin(p) >= kChunk; }
  __device__ __forceinline__ void next() { chunk += gridDim.x; }
};

// The coefficients of an item's step, looked up where the item is another than before.
template <int CAP>
__device__ __forceinline__ void of_item(AdamStep& step, unsigned& t, int& known, const AdamParams<CAP>& p, unsigned k, float lr) {
  if ((int)k == known) return;
  known = (int)k;
  const long long count = *p.item[k].step + 1;
  t = (unsigned)count;
  step.c1 = lr / -expm1f((float)((double)count * p.log_beta1));
  step.c2 = rsqrtf(-expm1f((float)((double)count * p.log_beta2)));
}

// The last block to get here counts the steps, once nobody reads them any more.
template <int CAP>
__device__ __forceinline__ void count_steps(const AdamParams<CAP>& p) {
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicInc(p.ticket, gridDim.x - 1) == gridDim.x - 1;      // (back to 0 for the next launch)
  }
  __syncthreads();
  if (last)
    for (unsigned j = threadIdx.x; j < p.items; j += kAdamThreads) ++*p.item[j].step;
}

template <typename T, bool MASTER, int CAP>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamParams<CAP> p) {
  const float factor = p.factor ? *p.factor : 1.f;
  if (factor != factor) return;                // gradients that are no numbers: everything stays as it is
  const float lr = p.lr_at ? *p.lr_at : p.lr;
  AdamStep step{factor, p.beta1, p.beta2, p.one_less1, p.one_less2, p.eps, lr * p.decay, p.one, 0.f, 0.f};
  unsigned t = 0;
  int known = -1;
  for (Cursor<CAP> c; c.there(p); c.next()) {
    of_item(step, t, known, p, c.k, lr);
    if (c.whole(p)) turns<T, 32, MASTER, true>(step, p.item[c.k], c.begin(p), kChunk, true, p.keys, t);
    else turns<T, 32, MASTER, false>(step, p.item[c.k], c.begin(p), p.item[c.k].n - c.begin(p), c.wide(p), p.keys, t);
  }
  count_steps(p);
}

// 8 bits: what a turn needs comes into shared memory kStages - 1 turns ahead, every thread's own by itself (in registers it would cost
// the warps that hide the arithmetic).
constexpr int kStages = 4;
template <typename T, bool MASTER>
struct AdamStage {
  static constexpr int NG = sizeof(T) / 2, NX = MASTER ? 2 : NG;
  uint4 g[NG][kAdamThreads], x[NX][kAdamThreads];
  uint2 m[kAdamThreads], u[kAdamThreads];
  float scale[2][kAdamThreads / 32];
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const unsigned a = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(a), "l"(from), "n"(BYTES) : "memory");
}

// (Three blocks an SM with the stages of 16-bit weights.  Those of fp32 weights are 82 KB, so that two fit, with registers for three.)
template <typename T, bool MASTER, int CAP>
__global__ void __launch_bounds__(kAdamThreads, 3) adamw8_kernel(const __grid_constant__ AdamParams<CAP> p) {
  extern __shared__ uint4 s_raw[];
  using Stage = AdamStage<T, MASTER>;
  using X = std::conditional_t<MASTER, float, T>;
  Stage* stages = reinterpret_cast<Stage*>(s_raw);
  const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float factor = p.factor ? *p.factor : 1.f;
  if (factor != factor) return;
  const float lr = p.lr_at ? *p.lr_at : p.lr;
  AdamStep step{factor, p.beta1, p.beta2, p.one_less1, p.one_less2, p.eps, lr * p.decay, p.one, 0.f, 0.f};
  unsigned t = 0;
  int known = -1;
  // the fetching side: whole chunks alone
  Cursor<CAP> f;
  int f_at = 0, f_stage = 0;
  const T* f_grad = nullptr;
  const X* f_x = nullptr;
  const uint8_t *f_m = nullptr, *f_u = nullptr;
  const float* f_scale = nullptr;              // lane 0: m's, lane 1: the root's
  auto f_open = [&] {                          // the next whole chunk from here on
    while (f.there(p) && !f.whole(p)) f.next();
    if (f.chunk >= p.chunks) return;
    const AdamItem& a = p.item[f.k];
    const long long i = f.begin(p) + tid * 8;
    f_grad = static_cast<const T*>(a.grad) + i;
    f_x = (MASTER ? reinterpret_cast<const X*>(a.master) : static_cast<const X*>(a.param)) + i;
    f_m = static_cast<const uint8_t*>(a.m) + i;
    f_u = static_cast<const uint8_t*>(a.v) + i;
    f_scale = (lane ? a.v_scale : a.m_scale) + i / 256;
  };
  auto fetch = [&] {
    if (f.chunk < p.chunks) {
      Stage& s = stages[f_stage];
#pragma unroll
      for (int k = 0; k < Stage::NG; ++k) copy_async<16>(&s.g[k][tid], reinterpret_cast<const uint4*>(f_grad) + k);
#pragma unroll
      for (int k = 0; k < Stage::NX; ++k) copy_async<16>(&s.x[k][tid], reinterpret_cast<const uint4*>(f_x) + k);
      copy_async<8>(&s.m[tid], f_m);
      copy_async<8>(&s.u[tid], f_u);
      if (lane < 2) copy_async<4>(&s.scale[lane][warp], f_scale);
      f_grad += kTurn; f_x += kTurn; f_m += kTurn; f_u += kTurn; f_scale += kTurn / 256;
      f_at += kTurn;
      if (f_at == kChunk) {
        f_at = 0;
        f.next();
        f_open();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    f_stage = f_stage + 1 == kStages ? 0 : f_stage + 1;
  };
  f_open();
#pragma unroll
  for (int k = 0; k + 1 < kStages; ++k) fetch();
  int stage = 0;
  for (Cursor<CAP> c; c.there(p); c.next()) {
    of_item(step, t, known, p, c.k, lr);
    const AdamItem& a = p.item[c.k];
    if (!c.whole(p)) {
      turns<T, 8, MASTER, false>(step, a, c.begin(p), a.n - c.begin(p), c.wide(p), p.keys, t);
      continue;
    }
    const long long i0 = c.begin(p) + tid * 8;
    T* param = static_cast<T*>(a.param) + i0;
    float* master = MASTER ? a.master + i0 : nullptr;
    uint8_t *mb = static_cast<uint8_t*>(a.m) + i0, *ub = static_cast<uint8_t*>(a.v) + i0;
    float* scale = (lane ? a.v_scale : a.m_scale) + i0 / 256;
    unsigned long long block = (unsigned long long)i0 / 4;
#pragma unroll 1
    for (int at = 0; at < kChunk; at += kTurn, block += kTurn / 4) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();                            // (the scales are other lanes' copies; and this stage's next copies come behind everybody's reads)
      Stage& s = stages[stage];
      stage = stage + 1 == kStages ? 0 : stage + 1;
      float ge[8], xe[8];
      Raw<T> g;
      Raw<X> x;
#pragma unroll
      for (int k = 0; k < Stage::NG; ++k) g.v[k] = s.g[k][tid];
#pragma unroll
      for (int k = 0; k < Stage::NX; ++k) x.v[k] = s.x[k][tid];
      uint2 m8 = s.m[tid], u8 = s.u[tid];
      float ms = s.scale[0][warp], us = s.scale[1][warp];
      g.get(ge);
      x.get(xe);
      fetch();
      step(ge, m8, u8, ms, us, xe, [&](int h, unsigned (&w)[4]) { draw4(w, p.keys, block + h, t, a.number); });
      store8_bytes<true>(mb + at, 8, true, m8);
      store8_bytes<true>(ub + at, 8, true, u8);
      if (lane < 2) scale[at / 256] = lane ? us : ms;
      if constexpr (MASTER) store8<true>(master + at, 8, true, xe);
      store8<true>(param + at, 8, true, xe);
    }
  }
  count_steps(p);
}

// ---------------------------------------------------------------- the norm of all gradients
struct NormItem {
  const void* grad;
  long long n;
  unsigned first;
  int dtype;                     // and 16 where the address is no multiple of 16
};
template <int CAP>
struct GradNormParams {
  NormItem item[CAP];
  unsigned items, chunks;
  double* partial;               // of this launch's blocks
  const double* all;             // of all launches' blocks, `blocks` of them: the last launch has them
  unsigned blocks;
  float max_norm;
  float* out;                    // norm, factor; null before the last launch
  unsigned* ticket;
};
constexpr int kNormChunk = 2 * kTurn;

template <typename T>
__device__ __forceinline__ double squares(const Raw<T>& raw) {
  float z[8];
  double t = 0;
  raw.get(z);
#pragma unroll
  for (int e = 0; e < 8; ++e) t = fma((double)z[e], (double)z[e], t);
  return t;
}
template <typename T>
__device__ __forceinline__ double chunk_squares(const T* g, long long i, long long n, bool wide) {
  constexpr int kParts = kNormChunk / kTurn;
  double sum = 0;
  if (wide && i - threadIdx.x * 8 + kNormChunk <= n) {
    Raw<T> raw[kParts];
#pragma unroll
    for (int part = 0; part < kParts; ++part) raw[part].template load<true>(g + i + part * kTurn, 8, true);
#pragma unroll
    for (int part = 0; part < kParts; ++part) sum += squares(raw[part]);
  } else {
#pragma unroll 1
    for (long long at = i; at < n && at < i + kNormChunk; at += kTurn) {
      Raw<T> raw;
      raw.template load<false>(g + at, n - at, wide);
      sum += squares(raw);
    }
  }
  return sum;
}

// In 64 bits throughout: the factor is the same whatever the order, but for one rounding to 32 bits.
template <int CAP>
__global__ void __launch_bounds__(kAdamThreads) grad_norm_kernel(const __grid_constant__ GradNormParams<CAP> p) {
  __shared__ double s[kAdamThreads / 32];
  __shared__ bool last;
  const unsigned tid = threadIdx.x;
  double sum = 0;
  unsigned k = 0;
  for (unsigned chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    while (k + 1 < p.items && chunk >= p.item[k + 1].first) ++k;
    const NormItem& a = p.item[k];
    const long long i = (long long)(chunk - a.first) * kNormChunk + tid * 8;
    const bool wide = !(a.dtype & 16);
    const int dtype = a.dtype & 15;
    sum += dtype == BLSTM_F32 ? chunk_squares(static_cast<const float*>(a.grad), i, a.n, wide)
         : dtype == BLSTM_F16 ? chunk_squares(static_cast<const __half*>(a.grad), i, a.n, wide)
                              : chunk_squares(static_cast<const __nv_bfloat16*>(a.grad), i, a.n, wide);
  }
  auto over_block = [&](double v) {            // in thread 0
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if ((tid & 31) == 0) s[tid / 32] = v;
    __syncthreads();
    if (tid == 0)
      for (int w = 1; w < kAdamThreads / 32; ++w) v += s[w];
    return v;
  };
  sum = over_block(sum);
  if (tid == 0) {
    p.partial[blockIdx.x] = sum;
    __threadfence();
    last = p.out && atomicInc(p.ticket, gridDim.x - 1) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum = 0;
  for (unsigned b = tid; b < p.blocks; b += kAdamThreads) sum += __ldcg(p.all + b);
  sum = over_block(sum);
  if (tid == 0) {
    const double norm = sqrt(sum);
    p.out[0] = (float)norm;
    const float f = (float)(p.max_norm / (norm + 1e-6));
    p.out[1] = isfinite(sum) ? fminf(f, 1.f) : __int_as_float(0x7fffffff);
  }
}

// ---------------------------------------------------------------- host
constexpr int kFew = 32, kMany = 384;          // tensors of a launch, with 2.7 and 31 KB of parameters

// (More blocks than an SM has at a time: SMs are not all as near to all memory, and blocks that are still to come even that out.  Of steps
// with 32 bits, 3, 4, 8, 16, 32 blocks an SM: 29.8 M bf16 weights with masters, clipped, 177, 183, 155, 151, 155 us.  With 8 bits a block
// fills its stages first, which fewer chunks for each make dearer: 151 M bf16 weights 403, 403, 391, 391, 392, 14 M fp32 ones with 8 and 16
// 80 and 85.  Norms of gradients with 4, 8, 16: the 29.8 M 151, 147, 149.)
constexpr unsigned kStepBlocks = 16, kFewBlocks = 8;
static unsigned adam_grid(unsigned chunks, unsigned each) { return std::min(chunks, each * (unsigned)plan_sm_count()); }

template <typename T, int BITS, bool MASTER, int CAP>
static int launch_adamw(const blstm_adamw_desc& d, const blstm_adamw_item* items, int n, cudaStream_t st) {
  AdamParams<CAP> p{};
  unsigned long long chunks = 0;
  for (int k = 0; k < n; ++k) {
    const blstm_adamw_item& s = items[k];
    AdamItem& a = p.item[k];
    a.param = s.param; a.grad = s.grad; a.m = s.exp_avg; a.v = s.exp_avg_sq;
    a.m_scale = s.exp_avg_scale; a.v_scale = s.exp_avg_sq_scale; a.master = s.master;
    a.step = reinterpret_cast<long long*>(s.step);
    a.n = s.n; a.first = (unsigned)chunks; a.number = s.number;
    if (aligned(16, s.param, s.grad, s.exp_avg, s.exp_avg_sq, s.master)) p.wide[k / 64] |= 1ull << k % 64;
    chunks += (unsigned long long)((s.n + kChunk - 1) / kChunk);
    if (chunks > INT32_MAX) return BLSTM_E_TOO_LARGE;
  }
  p.items = (unsigned)n; p.chunks = (unsigned)chunks;
  for (int r = 0; r < 10; ++r) {
    p.keys[2 * r] = (unsigned)d.seed + r * 0x9E3779B9u;
    p.keys[2 * r + 1] = (unsigned)(d.seed >> 32) + r * 0xBB67AE85u;
  }
  p.lr = (float)d.lr; p.beta1 = (float)d.beta1; p.beta2 = (float)d.beta2;
  p.one_less1 = (float)(1 - d.beta1); p.one_less2 = (float)(1 - d.beta2);
  p.eps = (float)d.eps; p.decay = (float)d.weight_decay;
  p.one = 1.f;
  p.log_beta1 = std::log(d.beta1); p.log_beta2 = std::log(d.beta2);
  p.lr_at = d.lr_at; p.factor = d.factor; p.ticket = d.ticket;
  if constexpr (BITS == 32) {
    adamw_kernel<T, MASTER, CAP><<<adam_grid(p.chunks, kStepBlocks), kAdamThreads, 0, st>>>(p);
  } else {
    constexpr int smem = kStages * (int)sizeof(AdamStage<T, MASTER>);
    if constexpr (smem > 48 * 1024) BLSTM_CUDA_OK(cudaFuncSetAttribute(adamw8_kernel<T, MASTER, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    adamw8_kernel<T, MASTER, CAP><<<adam_grid(p.chunks, kFewBlocks), kAdamThreads, smem, st>>>(p);
  }
  BLSTM_CUDA_OK(cudaGetLastError());
  count_launch();
  return BLSTM_OK;
}

template <typename T, int BITS, bool MASTER>
static int launch_adamw(const blstm_adamw_desc& d, cudaStream_t st) {
  for (int at = 0; at < d.items; at += kMany) {
    const int n = std::min(d.items - at, (int)kMany);
    const int rc = n <= kFew ? launch_adamw<T, BITS, MASTER, kFew>(d, d.item + at, n, st) : launch_adamw<T, BITS, MASTER, kMany>(d, d.item + at, n, st);
    if (rc) return rc;
  }
  return BLSTM_OK;
}

template <int CAP>
static int launch_grad_norm(const blstm_grad_norm_desc& d, int at, int n, unsigned& blocks, bool last, cudaStream_t st) {
  GradNormParams<CAP> p{};
  unsigned long long chunks = 0;
  for (int k = 0; k < n; ++k) {
    const blstm_grad_item& s = d.item[at + k];
    p.item[k] = {s.grad, (long long)s.n, (unsigned)chunks, s.dtype | (aligned(16, s.grad) ? 0 : 16)};
    chunks += (unsigned long long)((s.n + kNormChunk - 1) / kNormChunk);
    if (chunks > INT32_MAX) return BLSTM_E_TOO_LARGE;
  }
  const unsigned grid = adam_grid((unsigned)chunks, kFewBlocks);
  double* all = static_cast<double*>(d.workspace);
  p.items = (unsigned)n; p.chunks = (unsigned)chunks;
  p.partial = all + blocks; p.all = all;
  blocks += grid;
  p.blocks = blocks;
  p.max_norm = d.max_norm;
  p.out = last ? d.out : nullptr;
  p.ticket = d.ticket;
  grad_norm_kernel<CAP><<<grid, kAdamThreads, 0, st>>>(p);
  BLSTM_CUDA_OK(cudaGetLastError());
  count_launch();
  return BLSTM_OK;
}

}  // namespace blstm

using namespace blstm;

extern "C" {

int blstm_adamw(const blstm_adamw_desc* d, void* stream) {
  if (!d || !valid_dtype(d->dtype) || (d->bits != 32 && d->bits != 8) || d->items < 0 || (d->items && !d->item) || !(d->beta1 >= 0 && d->beta1 < 1) ||
      !(d->beta2 >= 0 && d->beta2 < 1) || !(d->eps == 0 || d->eps >= FLT_MIN) || !std::isfinite((float)d->eps) || !std::isfinite((float)d->weight_decay) ||
      (!d->lr_at && !std::isfinite((float)d->lr)) || !aligned(4, d->lr_at, d->factor, d->ticket) || !d->ticket)
    return BLSTM_E_INVALID_ARG;
  const size_t e = dtype_bytes(d->dtype), se = d->bits == 32 ? 4 : 1;
  const bool master = d->items && d->item[0].master;
  if (master && d->dtype == BLSTM_F32) return BLSTM_E_INVALID_ARG;
  for (int k = 0; k < d->items; ++k) {
    const blstm_adamw_item& s = d->item[k];
    if (s.n <= 0 || !s.param || !s.grad || !s.exp_avg || !s.exp_avg_sq || !s.step || (s.master != nullptr) != master || !aligned(e, s.param, s.grad) ||
        !aligned(se, s.exp_avg, s.exp_avg_sq) || !aligned(4, s.master, s.exp_avg_scale, s.exp_avg_sq_scale) || !aligned(8, s.step) ||
        (d->bits == 8 && (!s.exp_avg_scale || !s.exp_avg_sq_scale)))
      return BLSTM_E_INVALID_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2)
      if (master) return d->bits == 32 ? launch_adamw<T, 32, true>(*d, st) : launch_adamw<T, 8, true>(*d, st);
    return d->bits == 32 ? launch_adamw<T, 32, false>(*d, st) : launch_adamw<T, 8, false>(*d, st);
  });
}

size_t blstm_grad_norm_workspace(int items) {
  return items <= 0 ? 256 : round_up((size_t)((items + kMany - 1) / kMany) * adam_grid(UINT32_MAX, kFewBlocks) * sizeof(double), 256);
}

int blstm_grad_norm(const blstm_grad_norm_desc* d, void* stream) {
  if (!d || d->items < 0 || (d->items && !d->item) || !(d->max_norm > 0.f) || !d->out || !d->ticket || !aligned(4, d->out, d->ticket)) return BLSTM_E_INVALID_ARG;
  for (int k = 0; k < d->items; ++k)
    if (!valid_dtype(d->item[k].dtype) || d->item[k].n <= 0 || !d->item[k].grad || !aligned(dtype_bytes(d->item[k].dtype), d->item[k].grad))
      return BLSTM_E_INVALID_ARG;
  if (!d->workspace || !aligned(256, d->workspace) || d->workspace_bytes < blstm_grad_norm_workspace(d->items)) return BLSTM_E_WORKSPACE;
  unsigned blocks = 0;
  for (int at = 0; at < d->items; at += kMany) {
    const int n = std::min(d->items - at, (int)kMany);
    const bool last = at + n == d->items;
    const int rc = n <= kFew ? launch_grad_norm<kFew>(*d, at, n, blocks, last, (cudaStream_t)stream)
                             : launch_grad_norm<kMany>(*d, at, n, blocks, last, (cudaStream_t)stream);
    if (rc) return rc;
  }
  return BLSTM_OK;
}

}  // extern "C"
