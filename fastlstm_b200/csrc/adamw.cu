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
#include <cmath>

#include "language.cuh"

namespace blstm {

constexpr int kChunk = 2048, kAdamThreads = 256;       // elements of a block's turn: 8 a thread, 256 (a scale) a warp

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
  float lr, beta1, beta2, one_less1, one_less2, eps, decay;
  double log_beta1, log_beta2;
  const float *lr_at, *factor;
  unsigned* ticket;
};

// Eight elements from i on as floats; those from n on are 0.
template <typename T>
__device__ __forceinline__ void load8(const T* p, long long i, long long n, bool wide, float (&z)[8]) {
  if (wide && i + 8 <= n) {
#pragma unroll
    for (int k = 0; k < 8; k += kPer<T>) unpack(*reinterpret_cast<const uint4*>(p + i + k), z + k, T{});
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] = i + k < n ? ld_f(p + i + k) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, long long i, long long n, bool wide, const float (&z)[8]) {
  if (wide && i + 8 <= n) {
#pragma unroll
    for (int k = 0; k < 8; k += kPer<T>) *reinterpret_cast<uint4*>(p + i + k) = pack(z + k, T{});
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[i + k] = Elem<T>::from_f(z[k]);
  }
}

// Eight e4m3 numbers as they lie in memory.
__device__ __forceinline__ uint2 load8_bytes(const uint8_t* p, long long i, long long n, bool wide) {
  if (wide && i + 8 <= n) return *reinterpret_cast<const uint2*>(p + i);
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (i + k < n) w[k / 4] |= (unsigned)p[i + k] << k % 4 * 8;
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store8_bytes(uint8_t* p, long long i, long long n, bool wide, uint2 w) {
  if (wide && i + 8 <= n) {
    *reinterpret_cast<uint2*>(p + i) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[i + k] = (uint8_t)((k < 4 ? w.x : w.y) >> k % 4 * 8);
  }
}
__device__ __forceinline__ void decode8(uint2 w, float scale, float (&z)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const unsigned short two = (unsigned short)((k < 4 ? w.x : w.y) >> k % 4 * 8);
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    z[k] = f.x * scale;
    z[k + 1] = f.y * scale;
  }
}

// A magnitude of at most 448 as an e4m3 number, in bits 20 to 27: times 2^-120 its bits are the top bits of the float's, subnormal
// numbers too, and adding `chance` (20 bits) below them rounds up with the probability of what is cut off.
__device__ __forceinline__ unsigned encode(float magnitude, unsigned chance) {
  return min(__float_as_uint(magnitude * 0x1p-120f) + chance, (127u << 20) - 1);
}

// The words of elements 4 block .. 4 block + 7 in step t of tensor `number`: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) with the seed
// as the key and (block, t, number) as the counter.
__device__ __forceinline__ void draw8(unsigned (&w)[8], const unsigned* keys, unsigned long long block, unsigned t, unsigned number) {
#pragma unroll
  for (int b = 0; b < 8; b += 4) {
    const unsigned long long c = block + b / 4;
    w[b] = (unsigned)c;
    w[b + 1] = (unsigned)(c >> 32);
    w[b + 2] = t;
    w[b + 3] = number;
  }
#pragma unroll
  for (int r = 0; r < 10; ++r) {
#pragma unroll
    for (int b = 0; b < 8; b += 4) {
      const unsigned long long x = (unsigned long long)w[b] * 0xD2511F53u, y = (unsigned long long)w[b + 2] * 0xCD9E8D57u;
      w[b] = (unsigned)(y >> 32) ^ w[b + 1] ^ keys[2 * r];
      w[b + 1] = (unsigned)y;
      w[b + 2] = (unsigned)(x >> 32) ^ w[b + 3] ^ keys[2 * r + 1];
      w[b + 3] = (unsigned)x;
    }
  }
}

// The largest magnitude of a warp's numbers: the bits of magnitudes have their order, and NaN comes last.
__device__ __forceinline__ float warp_most(const float (&z)[8]) {
  unsigned most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(z[e]) & 0x7fffffffu);
  return __uint_as_float(__reduce_max_sync(~0u, most));
}
// The codes of four numbers in their order in memory, from the bits 20 to 27 of four words.
__device__ __forceinline__ unsigned bytes_of(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a << 4, b << 4, 0x0073), __byte_perm(c << 4, d << 4, 0x0073), 0x5410);
}
__device__ __forceinline__ unsigned signs_of(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0073), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0073), 0x5410) & 0x80808080u;
}
__device__ __forceinline__ float reciprocal_fast(float x) {      // to 2^-23
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sqrt_fast(float x) {      // to 2^-22
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a scale and its inverse are for a largest magnitude; magnitudes below 2^-110 are 0 (the inverse would not be a number of 32 bits).
struct Scale {
  float up, down;
  __device__ __forceinline__ explicit Scale(float most)
      : up(most > 0x1p-110f ? 1.f / most * 448.f : 0.f), down(most <= 0x1p-110f ? 0.f : most * (1.f / 448.f)) {}
};

template <typename T, int BITS, bool MASTER, int CAP>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamParams<CAP> p) {
  const unsigned tid = threadIdx.x, lane = tid & 31;
  const float factor = p.factor ? *p.factor : 1.f;
  if (factor != factor) return;                // gradients that are no numbers: everything stays as it is
  unsigned k = 0, t = 0;
  int known = -1;                              // the item that t, c1 and c2 are of
  float c1 = 0.f, c2 = 0.f;
  const float lr = p.lr_at ? *p.lr_at : p.lr, decay = lr * p.decay;
  for (unsigned chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    while (k + 1 < p.items && chunk >= p.item[k + 1].first) ++k;
    const AdamItem& a = p.item[k];
    const bool wide = p.wide[k / 64] >> k % 64 & 1;
    const long long i = (long long)(chunk - a.first) * kChunk + tid * 8;
    float g[8], m[8], v[8], x[8];
    uint2 m8, v8;
    float m_scale, v_scale;
    const long long block = i / 256;           // (of a warp)
    load8(static_cast<const T*>(a.grad), i, a.n, wide, g);
    if constexpr (BITS == 32) {
      load8(static_cast<const float*>(a.m), i, a.n, wide, m);
      load8(static_cast<const float*>(a.v), i, a.n, wide, v);
    } else {
      m8 = load8_bytes(static_cast<const uint8_t*>(a.m), i, a.n, wide);
      v8 = load8_bytes(static_cast<const uint8_t*>(a.v), i, a.n, wide);
      m_scale = block * 256 < a.n ? a.m_scale[block] : 0.f;
      v_scale = block * 256 < a.n ? a.v_scale[block] : 0.f;
    }
    if constexpr (MASTER) load8(a.master, i, a.n, wide, x);
    else load8(static_cast<const T*>(a.param), i, a.n, wide, x);
    if ((int)k != known) {
      known = (int)k;
      const long long count = *a.step + 1;
      t = (unsigned)count;
      c1 = lr / -expm1f((float)((double)count * p.log_beta1));
      c2 = rsqrtf(-expm1f((float)((double)count * p.log_beta2)));
    }
    if constexpr (BITS == 8) {
      decode8(m8, m_scale, m);
      decode8(v8, v_scale, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= v[e];
    }
    float u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = g[e] * factor;
      if constexpr (BITS == 32) {
        m[e] = fmaf(p.beta1, m[e], p.one_less1 * ge);
        v[e] = fmaf(p.beta2, v[e], p.one_less2 * (ge * ge));
        u[e] = sqrt_fast(v[e]);
      } else {
        // (each operation rounded by itself, so that what is rounded to 8 bits depends on the formula alone)
        m[e] = __fadd_rn(__fmul_rn(p.beta1, m[e]), __fmul_rn(p.one_less1, ge));
        u[e] = __fsqrt_rn(__fadd_rn(__fmul_rn(p.beta2, v[e]), __fmul_rn(p.one_less2, __fmul_rn(ge, ge))));
      }
      x[e] -= fmaf(decay, x[e], c1 * m[e] * reciprocal_fast(fmaf(u[e], c2, p.eps)));
    }
    if constexpr (MASTER) store8(a.master, i, a.n, wide, x);
    store8(static_cast<T*>(a.param), i, a.n, wide, x);
    if constexpr (BITS == 32) {
      store8(static_cast<float*>(a.m), i, a.n, wide, m);
      store8(static_cast<float*>(a.v), i, a.n, wide, v);
    } else {
      const Scale sm(warp_most(m)), su(warp_most(u));
      unsigned w[8], cm[8], cu[8];
      draw8(w, p.keys, (unsigned long long)i / 4, t, a.number);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cm[e] = encode(fabsf(m[e]) * sm.up, w[e] << 4 & 0xffff0u);
        cu[e] = encode(u[e] * su.up, w[e] >> 12 & 0xffff0u);
        if (u[e] * su.up > 0.f) cu[e] = max(cu[e], 1u << 20);
      }
      store8_bytes(static_cast<uint8_t*>(a.m), i, a.n, wide, make_uint2(bytes_of(cm[0], cm[1], cm[2], cm[3]) | signs_of(m[0], m[1], m[2], m[3]),
                                                                        bytes_of(cm[4], cm[5], cm[6], cm[7]) | signs_of(m[4], m[5], m[6], m[7])));
      store8_bytes(static_cast<uint8_t*>(a.v), i, a.n, wide, make_uint2(bytes_of(cu[0], cu[1], cu[2], cu[3]), bytes_of(cu[4], cu[5], cu[6], cu[7])));
      if (lane == 0 && block * 256 < a.n) {
        a.m_scale[block] = sm.down;
        a.v_scale[block] = su.down;
      }
    }
  }
  // The last block to get here counts the steps, once nobody reads them any more.
  __shared__ bool last;
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    last = atomicInc(p.ticket, gridDim.x - 1) == gridDim.x - 1;      // (back to 0 for the next launch)
  }
  __syncthreads();
  if (last)
    for (unsigned j = tid; j < p.items; j += kAdamThreads) ++*p.item[j].step;
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
constexpr int kNormChunk = 4 * kChunk;

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* g, long long i, long long n, bool wide) {
  double sum = 0;
#pragma unroll
  for (int part = 0; part < kNormChunk / kChunk; ++part) {
    float z[8], t = 0.f;
    load8(g, i + part * kChunk, n, wide, z);
#pragma unroll
    for (int e = 0; e < 8; ++e) t = fmaf(z[e], z[e], t);
    sum += t;
  }
  return sum;
}

// Squares of eight neighbours are added up in 32 bits, what they come to in 64.
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

static unsigned adam_grid(unsigned chunks) { return std::min(chunks, 8u * (unsigned)plan_sm_count()); }

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
  p.log_beta1 = std::log(d.beta1); p.log_beta2 = std::log(d.beta2);
  p.lr_at = d.lr_at; p.factor = d.factor; p.ticket = d.ticket;
  adamw_kernel<T, BITS, MASTER, CAP><<<adam_grid(p.chunks), kAdamThreads, 0, st>>>(p);
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
  const unsigned grid = adam_grid((unsigned)chunks);
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
      !(d->beta2 >= 0 && d->beta2 < 1) || !(d->eps >= 0 && std::isfinite((float)d->eps)) || !std::isfinite((float)d->weight_decay) ||
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
  return items <= 0 ? 256 : round_up((size_t)((items + kMany - 1) / kMany) * adam_grid(UINT32_MAX) * sizeof(double), 256);
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
