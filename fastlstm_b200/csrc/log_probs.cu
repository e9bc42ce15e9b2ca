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
  unsigned n, vocab;
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

// The order of top alternatives: larger logits first (NaN before all), then lower numbers.  Never 0.
__device__ __forceinline__ unsigned value_key(float z) {
  if (z != z) return 0xffffffffu;
  const unsigned b = __float_as_uint(z + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_key(float z, unsigned j) { return (unsigned long long)value_key(z) << 32 | (0xffffffffu - j); }

// A part of a row: its maximum, sum of 2^(d) and of d 2^(d), d = distance from the maximum in powers of two.
struct Part {
  float m, s, t;
  __device__ __forceinline__ void add(const Part& o, float to_log2) {
    const float M = max_nan(m, o.m);
    const float a = max_nan((m - M) * to_log2, kFar), b = max_nan((o.m - M) * to_log2, kFar);
    const float fa = exp2f(a), fb = exp2f(b);
    t = fa * (t + s * a) + fb * (o.t + o.s * b);
    s = fa * s + fb * o.s;
    m = M;
  }
};

template <typename T>
__global__ void __launch_bounds__(256) score_kernel(const __grid_constant__ ScoreParams p) {
  __shared__ Part s_part[8];
  __shared__ unsigned long long s_key[8];
  const unsigned r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long token = p.tokens(r);
  if (token == p.ignore) {
    if (tid == 0) {
      p.log_probs[r] = 0.f;
      p.entropy[r] = 0.f;
      for (int i = 0; i < 3; ++i) p.stats[(size_t)i * p.n + r] = 0.f;
    }
    if (tid < (unsigned)p.top) {
      p.top_log_probs[(size_t)r * p.top + tid] = -INFINITY;
      p.top_tokens[(size_t)r * p.top + tid] = -1;
    }
    return;
  }
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  Part a{kLowest, 0.f, 0.f};
  for (unsigned j = tid; j < p.vocab; j += 256) {
    const float z = ld_f(row + j);
    if (!(z <= a.m)) a.add(Part{z, 1.f, 0.f}, p.to_log2);
    else {
      const float d = max_nan((z - a.m) * p.to_log2, kFar), e = exp2f(d);
      a.s += e;
      a.t += e * d;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) a.add(Part{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.t, o)}, p.to_log2);
  if (lane == 0) s_part[warp] = a;
  __syncthreads();
  a = s_part[0];
  for (int w = 1; w < 8; ++w) a.add(s_part[w], p.to_log2);
  const bool none = a.s == 0.f;               // every logit is -inf
  const float log2s = log2f(a.s);
  auto lp = [&](float z) { return none ? -INFINITY : (z - a.m) * p.per_temperature - log2s * kLn2; };
  if (tid == 0) {
    const bool in = token >= 0 && token < p.vocab;
    const float h = none ? 0.f : (log2s - a.t / a.s) * kLn2;
    p.log_probs[r] = in ? lp(ld_f(row + token)) : __int_as_float(0x7fffffff);
    p.entropy[r] = h;
    p.stats[r] = a.m; p.stats[(size_t)p.n + r] = log2s; p.stats[2 * (size_t)p.n + r] = h;
    if (!in) report_token(p.mailbox, r, token);
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
    for (unsigned j = tid; j < p.vocab; j += 256) {
      const unsigned long long q = order_key(ld_f(row + j), j);
      if (q < last && q > best) best = q;
    }
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
    __syncthreads();
    if (lane == 0) s_key[warp] = best;
    __syncthreads();
    for (int w = 0; w < 8; ++w) best = max(best, s_key[w]);
    last = best;
    if (tid == 0) {
      const unsigned j = 0xffffffffu - (unsigned)best;
      p.top_log_probs[(size_t)r * p.top + k] = lp(ld_f(row + j));
      p.top_tokens[(size_t)r * p.top + k] = j;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) score_grad_kernel(const __grid_constant__ ScoreParams p) {
  const unsigned r = blockIdx.x;
  const long long token = p.tokens(r);
  const T* row = static_cast<const T*>(p.logits) + p.rows(r);
  T* out = static_cast<T*>(p.dlogits) + p.drows(r);
  const float m = p.stats[r], log2s = p.stats[(size_t)p.n + r], h = p.stats[2 * (size_t)p.n + r];
  if (token == p.ignore || log2s == -INFINITY) {
    for (unsigned j = threadIdx.x; j < p.vocab; j += 256) out[j] = Elem<T>::from_f(0.f);
    return;
  }
  const float g_lp = p.g_lp && token >= 0 && token < p.vocab ? p.g_lp[p.g_lp_map(r)] : 0.f, g_h = p.g_h ? p.g_h[p.g_h_map(r)] : 0.f;
  float g = g_lp;
  if (p.g_top)
    for (int k = 0; k < p.top; ++k) g += p.g_top[(size_t)r * p.top + k];
  const float a = g + g_h * h, b = g_h * kLn2;
  for (unsigned j = threadIdx.x; j < p.vocab; j += 256) {
    const float d = max_nan((ld_f(row + j) - m) * p.to_log2, kFar) - log2s;
    float v = -exp2f(d) * (a + b * d);
    if (j == token) v += g_lp;
    if (p.g_top)
      for (int k = 0; k < p.top; ++k)
        if (p.top_tokens[(size_t)r * p.top + k] == j) v += p.g_top[(size_t)r * p.top + k];
    out[j] = Elem<T>::from_f(v * p.per_temperature);
  }
}

static int check_score(const blstm_score_desc* d, const void* logits, const void* tokens) {
  if (!d || !valid_dtype(d->dtype) || (d->token_bits != 32 && d->token_bits != 64) || !valid_rows(d->n0, d->n1) || d->vocab <= 0 ||
      d->vocab >= INT32_MAX || d->top < 0 || d->top > BLSTM_MAX_TOP || d->top > d->vocab || !(d->temperature >= 1e-30f && d->temperature < INFINITY))
    return BLSTM_E_INVALID_ARG;
  if (d->n0 && d->n1 && (!logits || !tokens || reinterpret_cast<uintptr_t>(logits) % dtype_bytes(d->dtype))) return BLSTM_E_INVALID_ARG;
  return BLSTM_OK;
}

static ScoreParams score_params(const blstm_score_desc& d, const void* logits, const void* tokens) {
  ScoreParams p{};
  p.logits = logits;
  p.rows = row_map(d.n1, d.logits_stride);
  p.tokens = {tokens, row_map(d.n1, d.token_stride), d.token_bits == 64};
  p.ignore = d.ignore;
  p.n = (unsigned)(d.n0 * d.n1); p.vocab = (unsigned)d.vocab; p.top = d.top;
  p.per_temperature = (float)(1.0 / d.temperature);
  p.to_log2 = (float)(1.4426950408889634 / d.temperature);
  return p;
}

}  // namespace blstm

using namespace blstm;

extern "C" {

int blstm_token_log_probs(const blstm_score_desc* d, const void* logits, const void* tokens, float* log_probs, float* entropy,
                          float* top_log_probs, int64_t* top_tokens, float* stats, void* stream) {
  if (int rc = check_score(d, logits, tokens)) return rc;
  if (d->n0 == 0 || d->n1 == 0) return BLSTM_OK;
  if (!log_probs || !entropy || !stats || (d->top && (!top_log_probs || !top_tokens))) return BLSTM_E_INVALID_ARG;
  ScoreParams p = score_params(*d, logits, tokens);
  p.log_probs = log_probs; p.entropy = entropy; p.stats = stats;
  p.top_log_probs = top_log_probs; p.top_tokens = reinterpret_cast<long long*>(top_tokens);
  p.mailbox = current_mailbox();
  return with_type(d->dtype, [&](auto t) -> int {
    score_kernel<decltype(t)><<<p.n, 256, 0, (cudaStream_t)stream>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}

int blstm_token_log_probs_grad(const blstm_score_desc* d, const void* logits, const void* tokens, const float* stats, const int64_t* top_tokens,
                               const float* g_log_probs, const int64_t g_log_probs_stride[2], const float* g_entropy,
                               const int64_t g_entropy_stride[2], const float* g_top, void* dlogits, const int64_t dlogits_stride[2],
                               void* stream) {
  if (int rc = check_score(d, logits, tokens)) return rc;
  if (d->n0 == 0 || d->n1 == 0) return BLSTM_OK;
  if (!stats || !dlogits || !dlogits_stride || (g_log_probs && !g_log_probs_stride) || (g_entropy && !g_entropy_stride) || (g_top && (!top_tokens || d->top == 0)) ||
      ((reinterpret_cast<uintptr_t>(dlogits) - reinterpret_cast<uintptr_t>(logits)) & 15u) ||
      (d->n0 > 1 && ((dlogits_stride[0] - d->logits_stride[0]) * dtype_bytes(d->dtype) & 15)) ||
      (d->n1 > 1 && ((dlogits_stride[1] - d->logits_stride[1]) * dtype_bytes(d->dtype) & 15)))
    return BLSTM_E_INVALID_ARG;
  ScoreParams p = score_params(*d, logits, tokens);
  p.dlogits = dlogits;
  p.drows = row_map(d->n1, dlogits_stride);
  p.stats = const_cast<float*>(stats);
  p.top_tokens = reinterpret_cast<long long*>(const_cast<int64_t*>(top_tokens));
  p.g_lp = g_log_probs; p.g_h = g_entropy; p.g_top = g_top;
  if (g_log_probs) p.g_lp_map = row_map(d->n1, g_log_probs_stride);
  if (g_entropy) p.g_h_map = row_map(d->n1, g_entropy_stride);
  return with_type(d->dtype, [&](auto t) -> int {
    score_grad_kernel<decltype(t)><<<p.n, 256, 0, (cudaStream_t)stream>>>(p);
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}

}  // extern "C"
