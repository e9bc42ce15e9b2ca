// Root-mean-square norm of a sum of two tensors, and its gradient.
//
//   h = round(x + r)     i = 1 / sqrt(mean_j h_j^2 + eps)     y_j = h_j i w_j
//   n = dy w    dx = dr = i (n - h i^2 mean_j(n_j h_j)) + dh    dw_j = sum over the rows of dy_j h_j i
//
// The norm is of h as it is stored, so that backward, which reads h again, has the same numbers.  An output in 8 bits is
// q_j = e4m3(y_j / s), s = max_j |y_j| / 448, from y in 32 bits.  Bound by memory: forward reads x and r and writes h and y, backward
// reads h, dy and dh and writes dx; a row stays in the registers of the threads that share it.  Everything is added up in 32 bits.
#include <cuda_fp8.h>

#include <algorithm>

#include "language.cuh"

namespace blstm {

struct NormParams {
  const void *x, *r, *w, *dy;    // x: h in the gradient; r: dh there
  RowMap x_map, r_map, dy_map;
  void *y, *h;                   // y: dx in the gradient
  uint8_t* q;
  float *scales, *rstd, *dw;     // dw: the blocks' parts [parts][width], or the result where one block has all rows
  unsigned n, width, parts;
  bool x_alike, r_alike, dy_alike;       // rows on the same addresses modulo 16 as those of the results
  float eps, per_width;
};

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Two numbers as e4m3 ones, the first in the low byte.
__device__ __forceinline__ unsigned e4m3_two(float a, float b) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

// What a row is multiplied by, and its scale, from its largest magnitude.  (A product with 448 / most in place of a quotient by the scale for
// every element: a number within 2^-23 of the border between two of e4m3 may become the other one.  At most 2^-110 counts as 0: 448 over it would pass the largest
// float soon after, and the scale would lose its bits.)
__device__ __forceinline__ float row_up(float most) { return most > 0x1p-110f ? 448.f / most : 0.f; }
__device__ __forceinline__ float row_scale(float most) { return most <= 0x1p-110f ? 0.f : most / 448.f; }

__device__ __forceinline__ float abs_max(float m, float v) {      // NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}
struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct AbsMax {
  __device__ __forceinline__ float operator()(float a, float b) const { return abs_max(a, b); }
};

// A value over the G threads of a row, in each of them.  Groups of more than a warp are whole blocks; `s` has two sets of words that
// successive calls take in turn, so that one barrier a call does.
template <int G> constexpr int kWarps = G < 32 ? 1 : G / 32;
template <int G, typename F>
__device__ __forceinline__ float over_row(float v, float (*s)[kWarps<G>], unsigned& turn, F f) {
  const unsigned group = G < 32 ? ((1u << (G & 31)) - 1) << (threadIdx.x & 31 & ~(G - 1)) : ~0u;
#pragma unroll
  for (int o = G < 32 ? G / 2 : 16; o; o >>= 1) v = f(v, __shfl_xor_sync(group, v, o));
  if constexpr (G > 32) {
    float* w = s[turn & 1];
    ++turn;
    if ((threadIdx.x & 31) == 0) w[threadIdx.x / 32] = v;
    __syncthreads();
    v = w[threadIdx.x % (G / 32)];
#pragma unroll
    for (int o = G / 64; o; o >>= 1) v = f(v, __shfl_xor_sync(~0u, v, o));
  }
  return v;
}

// What a thread has of a row of `width` elements that G threads share in 16-byte pieces of the results: up to P of them, and where rows
// do not begin on a boundary (EDGES) one of the elements in front of the first piece and behind the last.  The threads' pieces are
// neighbours.  A group's rows are a multiple of eight apart, so all of them begin alike: what belongs to columns stays in registers.
template <typename T, int G, bool EDGES>
struct Cut {
  unsigned head, pieces, edges, at;
  __device__ __forceinline__ Cut(unsigned row, unsigned width) : at(threadIdx.x % G) {
    const unsigned off = (unsigned)((size_t)row * width % kPer<T>);      // of results that begin on a boundary
    head = EDGES ? min(width, (kPer<T> - off) % kPer<T>) : 0;
    pieces = (width - head) / kPer<T>;
    edges = EDGES ? width - pieces * kPer<T> : 0;
  }
  __device__ __forceinline__ bool has(int u) const { return u * G + at < pieces; }
  __device__ __forceinline__ unsigned first(int u) const { return head + (u * G + at) * kPer<T>; }
  __device__ __forceinline__ bool has_edge() const { return EDGES && at < edges; }
  __device__ __forceinline__ unsigned edge() const { return at < head ? at : at + pieces * kPer<T>; }
};

// A piece from anywhere: in one load where it lies on a boundary, else in narrow ones.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* p, bool whole) {
  if (whole) return load_stream(reinterpret_cast<const uint4*>(p));
  uint4 v;
  if (sizeof(T) == 4 || (reinterpret_cast<uintptr_t>(p) & 3) == 0) {
    const unsigned* w = reinterpret_cast<const unsigned*>(p);
    v = make_uint4(__ldg(w), __ldg(w + 1), __ldg(w + 2), __ldg(w + 3));
  } else {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    unsigned w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __ldg(h + 2 * k) | (unsigned)__ldg(h + 2 * k + 1) << 16;
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
template <typename T, int P, typename C>
__device__ __forceinline__ void load_row(uint4 (&v)[P], const T* row, const C& c, bool whole) {
#pragma unroll
  for (int u = 0; u < P; ++u) v[u] = c.has(u) ? load_piece(row + c.first(u), whole) : make_uint4(0, 0, 0, 0);
}

template <typename T, int P, int G, bool EDGES>
__global__ void __launch_bounds__(G < 128 ? 128 : G, G < 128 ? (P <= 2 ? 8 : 1) : G == 128 ? (P <= 2 ? 8 : 5) : 1) norm_kernel(const __grid_constant__ NormParams p) {
  constexpr int NT = G < 128 ? 128 : G, ROWS = NT / G, K = kPer<T>;
  __shared__ float s[2][kWarps<G>];
  unsigned turn = 0;
  const T* w = static_cast<const T*>(p.w);
  unsigned row = blockIdx.x * ROWS + threadIdx.x / G;
  const Cut<T, G, EDGES> c(row, p.width);
  uint4 weight[P];
  load_row(weight, w, c, !EDGES);
  const float edge_weight = c.has_edge() ? ld_f(w + c.edge()) : 0.f;
  for (; row < p.n; row += gridDim.x * ROWS) {
    const T* x = static_cast<const T*>(p.x) + p.x_map(row);
    uint4 v[P];
    float edge = 0.f, sum = 0.f;
    load_row(v, x, c, !EDGES || p.x_alike);
    if (c.has_edge()) edge = ld_f(x + c.edge());
    if (p.r) {
      const T* r = static_cast<const T*>(p.r) + p.r_map(row);
      T* h = static_cast<T*>(p.h) + (size_t)row * p.width;
      uint4 b[P];
      load_row(b, r, c, !EDGES || p.r_alike);
      if (c.has_edge()) {
        const T e = Elem<T>::from_f(edge + ld_f(r + c.edge()));
        h[c.edge()] = e;
        edge = Elem<T>::to_f(e);
      }
#pragma unroll
      for (int u = 0; u < P; ++u) {
        float z[K], o[K];
        unpack(v[u], z, T{});
        unpack(b[u], o, T{});
#pragma unroll
        for (int k = 0; k < K; ++k) z[k] += o[k];
        v[u] = pack(z, T{});
        if (c.has(u)) *reinterpret_cast<uint4*>(h + c.first(u)) = v[u];
      }
    }
#pragma unroll
    for (int u = 0; u < P; ++u) {
      float z[K];
      unpack(v[u], z, T{});
#pragma unroll
      for (int k = 0; k < K; ++k) sum = fmaf(z[k], z[k], sum);
    }
    sum = over_row<G>(fmaf(edge, edge, sum), s, turn, Add());
    const float i = rsqrtf(fmaf(sum, p.per_width, p.eps));
    if (p.rstd && c.at == 0) p.rstd[row] = i;
    auto normed = [&](int u, float (&z)[K]) {
      float o[K];
      unpack(v[u], z, T{});
      unpack(weight[u], o, T{});
#pragma unroll
      for (int k = 0; k < K; ++k) z[k] = z[k] * i * o[k];
    };
    edge = edge * i * edge_weight;
    if (p.q) {
      float most = fabsf(edge);
#pragma unroll
      for (int u = 0; u < P; ++u) {
        float z[K];
        normed(u, z);
#pragma unroll
        for (int k = 0; k < K; ++k) most = abs_max(most, z[k]);
      }
      most = over_row<G>(most, s, turn, AbsMax());
      const float up = row_up(most);
      uint8_t* q = p.q + (size_t)row * p.width;
      if (c.at == 0) p.scales[row] = row_scale(most);
#pragma unroll
      for (int u = 0; u < P; ++u) {
        if (!c.has(u)) continue;
        float z[K];
        normed(u, z);
        unsigned word[K / 4];
#pragma unroll
        for (int k = 0; k < K; k += 4) word[k / 4] = e4m3_two(z[k] * up, z[k + 1] * up) | e4m3_two(z[k + 2] * up, z[k + 3] * up) << 16;
        if constexpr (K == 8) *reinterpret_cast<uint2*>(q + c.first(u)) = make_uint2(word[0], word[K / 4 - 1]);
        else *reinterpret_cast<unsigned*>(q + c.first(u)) = word[0];
      }
      if (c.has_edge()) q[c.edge()] = (uint8_t)e4m3_two(edge * up, 0.f);
    } else {
      T* y = static_cast<T*>(p.y) + (size_t)row * p.width;
#pragma unroll
      for (int u = 0; u < P; ++u) {
        float z[K];
        normed(u, z);
        if (c.has(u)) *reinterpret_cast<uint4*>(y + c.first(u)) = pack(z, T{});
      }
      if (c.has_edge()) y[c.edge()] = Elem<T>::from_f(edge);
    }
  }
}

// (The sums stay in 32 bits: of 131072 rows a group has some 22, and sums in 64 bits would double the registers that hold them.  fp32, 627 x 301,
// all outputs together: 1.0e-7 off, where sums in 64 bits are 0.6e-7 off.)
// The gradient of the weight is added up over a group's rows in registers, over a block's groups in shared memory (a word of padding a
// piece, so that neighbours meet no bank twice), and over the blocks by sum_parts_kernel.
template <typename T, int P, int G, bool EDGES>
__global__ void __launch_bounds__(G < 128 ? 128 : G, G < 128 ? (P <= 2 ? 5 : 1) : G == 128 ? (P <= 2 ? 5 : 3) : 1) norm_grad_kernel(const __grid_constant__ NormParams p) {
  constexpr int NT = G < 128 ? 128 : G, ROWS = NT / G, K = kPer<T>, COLS = (P * G + (EDGES ? 1 : 0)) * K, PADDED = COLS / K * (K + 1);
  __shared__ float s[2][kWarps<G>];
  extern __shared__ float s_dw[];               // [ROWS][PADDED]
  unsigned turn = 0;
  const T* w = static_cast<const T*>(p.w);
  unsigned row = blockIdx.x * ROWS + threadIdx.x / G;
  const Cut<T, G, EDGES> c(row, p.width);
  uint4 weight[P];
  load_row(weight, w, c, !EDGES);
  const float edge_weight = c.has_edge() ? ld_f(w + c.edge()) : 0.f;
  float acc[P * K], edge_acc = 0.f;
#pragma unroll
  for (int k = 0; k < P * K; ++k) acc[k] = 0.f;
  for (; row < p.n; row += gridDim.x * ROWS) {
    const T *h = static_cast<const T*>(p.x) + p.x_map(row), *dy = static_cast<const T*>(p.dy) + p.dy_map(row);
    uint4 v[P], g[P], b[P];
    load_row(v, h, c, !EDGES || p.x_alike);
    load_row(g, dy, c, !EDGES || p.dy_alike);
    const float i = p.rstd[row];
    float h_edge = 0.f, g_edge = 0.f, b_edge = 0.f;
    if (c.has_edge()) {
      h_edge = ld_f(h + c.edge());
      g_edge = ld_f(dy + c.edge());
    }
    if (p.r) {
      const T* r = static_cast<const T*>(p.r) + p.r_map(row);
      load_row(b, r, c, !EDGES || p.r_alike);
      if (c.has_edge()) b_edge = ld_f(r + c.edge());
    } else {
#pragma unroll
      for (int u = 0; u < P; ++u) b[u] = make_uint4(0, 0, 0, 0);
    }
    auto weighed = [&](int u, float (&n)[K]) {         // dy w
      float o[K];
      unpack(g[u], n, T{});
      unpack(weight[u], o, T{});
#pragma unroll
      for (int k = 0; k < K; ++k) n[k] *= o[k];
    };
    edge_acc = fmaf(g_edge, h_edge * i, edge_acc);
    const float n_edge = g_edge * edge_weight;
    float sum = n_edge * h_edge;
#pragma unroll
    for (int u = 0; u < P; ++u) {
      float n[K], z[K], e[K];
      weighed(u, n);
      unpack(v[u], z, T{});
      unpack(g[u], e, T{});
#pragma unroll
      for (int k = 0; k < K; ++k) {
        sum = fmaf(n[k], z[k], sum);
        acc[u * K + k] = fmaf(e[k], z[k] * i, acc[u * K + k]);
      }
    }
    sum = over_row<G>(sum, s, turn, Add());
    const float by = sum * p.per_width * i * i;
    T* dx = static_cast<T*>(p.y) + (size_t)row * p.width;
#pragma unroll
    for (int u = 0; u < P; ++u) {
      float n[K], z[K], o[K];
      weighed(u, n);
      unpack(v[u], z, T{});
      unpack(b[u], o, T{});
#pragma unroll
      for (int k = 0; k < K; ++k) z[k] = fmaf(i, fmaf(-z[k], by, n[k]), o[k]);
      if (c.has(u)) *reinterpret_cast<uint4*>(dx + c.first(u)) = pack(z, T{});
    }
    if (c.has_edge()) dx[c.edge()] = Elem<T>::from_f(fmaf(i, fmaf(-h_edge, by, n_edge), b_edge));
  }
  if (!p.dw) return;
  auto cell = [&](unsigned j) -> float& { return s_dw[threadIdx.x / G * PADDED + j + j / K]; };
#pragma unroll
  for (int u = 0; u < P; ++u)
    if (c.has(u))
#pragma unroll
      for (int k = 0; k < K; ++k) cell(c.first(u) + k) = acc[u * K + k];
  if (c.has_edge()) cell(c.edge()) = edge_acc;
  __syncthreads();
  for (unsigned j = threadIdx.x; j < p.width; j += NT) {
    float t = s_dw[j + j / K];
#pragma unroll
    for (int k = 1; k < ROWS; ++k) t += s_dw[k * PADDED + j + j / K];
    if (p.parts > 1) p.dw[(size_t)blockIdx.x * p.width + j] = t;
    else reinterpret_cast<T*>(p.dw)[j] = Elem<T>::from_f(t);
  }
}

// Rows of any width and any strides, element by element: read again where they do not stay in registers.
template <typename T, int G>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_any_kernel(const __grid_constant__ NormParams p) {
  constexpr int ROWS = (G < 128 ? 128 : G) / G;
  __shared__ float s[2][kWarps<G>];
  unsigned turn = 0;
  const T* w = static_cast<const T*>(p.w);
  const unsigned at = threadIdx.x % G;
  for (unsigned row = blockIdx.x * ROWS + threadIdx.x / G; row < p.n; row += gridDim.x * ROWS) {
    const T* x = static_cast<const T*>(p.x) + p.x_map(row);
    float sum = 0.f;
    if (p.r) {
      const T* r = static_cast<const T*>(p.r) + p.r_map(row);
      T* h = static_cast<T*>(p.h) + (size_t)row * p.width;
#pragma unroll 4
      for (unsigned j = at; j < p.width; j += G) {
        const T e = Elem<T>::from_f(ld_f(x + j) + ld_f(r + j));
        h[j] = e;
        sum = fmaf(Elem<T>::to_f(e), Elem<T>::to_f(e), sum);
      }
      x = h;                                    // (what a thread has written itself)
    } else {
#pragma unroll 4
      for (unsigned j = at; j < p.width; j += G) sum = fmaf(ld_f(x + j), ld_f(x + j), sum);
    }
    sum = over_row<G>(sum, s, turn, Add());
    const float i = rsqrtf(fmaf(sum, p.per_width, p.eps));
    if (p.rstd && at == 0) p.rstd[row] = i;
    if (p.q) {
      float most = 0.f;
#pragma unroll 4
      for (unsigned j = at; j < p.width; j += G) most = abs_max(most, ld_f(x + j) * i * ld_f(w + j));
      most = over_row<G>(most, s, turn, AbsMax());
      const float up = row_up(most);
      if (at == 0) p.scales[row] = row_scale(most);
#pragma unroll 4
      for (unsigned j = at; j < p.width; j += G) p.q[(size_t)row * p.width + j] = (uint8_t)e4m3_two(ld_f(x + j) * i * ld_f(w + j) * up, 0.f);
    } else {
      T* y = static_cast<T*>(p.y) + (size_t)row * p.width;
#pragma unroll 4
      for (unsigned j = at; j < p.width; j += G) y[j] = Elem<T>::from_f(ld_f(x + j) * i * ld_f(w + j));
    }
  }
}

// (a thread has the same columns in every row, whose sums it keeps in the memory for its group's part)
template <typename T, int G>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_any_grad_kernel(const __grid_constant__ NormParams p) {
  constexpr int ROWS = (G < 128 ? 128 : G) / G;
  __shared__ float s[2][kWarps<G>];
  unsigned turn = 0;
  const T* w = static_cast<const T*>(p.w);
  const unsigned at = threadIdx.x % G, group = blockIdx.x * ROWS + threadIdx.x / G;
  float* part = p.dw ? p.dw + (size_t)group * p.width : nullptr;
  if (part)
    for (unsigned j = at; j < p.width; j += G) part[j] = 0.f;
  for (unsigned row = group; row < p.n; row += gridDim.x * ROWS) {
    const T *h = static_cast<const T*>(p.x) + p.x_map(row), *dy = static_cast<const T*>(p.dy) + p.dy_map(row);
    const float i = p.rstd[row];
    float sum = 0.f;
#pragma unroll 4
    for (unsigned j = at; j < p.width; j += G) {
      const float z = ld_f(h + j), e = ld_f(dy + j);
      sum = fmaf(e * ld_f(w + j), z, sum);
      if (part) part[j] = fmaf(e, z * i, part[j]);
    }
    sum = over_row<G>(sum, s, turn, Add());
    const float by = sum * p.per_width * i * i;
    const T* r = p.r ? static_cast<const T*>(p.r) + p.r_map(row) : nullptr;
    T* dx = static_cast<T*>(p.y) + (size_t)row * p.width;
#pragma unroll 4
    for (unsigned j = at; j < p.width; j += G)
      dx[j] = Elem<T>::from_f(fmaf(i, fmaf(-ld_f(h + j), by, ld_f(dy + j) * ld_f(w + j)), r ? ld_f(r + j) : 0.f));
  }
}

// dw = the sum of the parts, 32 columns a block, sixteen rows of them on their way to each of its warps (1480 parts of 512 columns with half the
// warps and eight rows 12.8 us, so 9; caches cold).
constexpr int kSumWarps = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kSumWarps) sum_parts_kernel(const float* parts, T* dw, unsigned n, unsigned width) {
  __shared__ float s[kSumWarps][33];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
  float t = 0.f;
  for (unsigned k0 = warp; k0 < n; k0 += 16 * kSumWarps) {
    float z[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) z[k] = j < width && k0 + k * kSumWarps < n ? __ldg(parts + (size_t)(k0 + k * kSumWarps) * width + j) : 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += z[k];
  }
  s[warp][lane] = t;
  __syncthreads();
  // a warp has a column, whose parts its lanes hold
  t = s[lane][warp];
#pragma unroll
  for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
  if (lane == 0 && blockIdx.x * 32 + warp < width) dw[blockIdx.x * 32 + warp] = Elem<T>::from_f(t);
}

// ---------------------------------------------------------------- host
// How a problem is cut: G threads a row with `pieces` 16-byte pieces each, or element by element (pieces 0); rows in edges and pieces
// where they do not begin on a boundary.
struct NormPlan {
  int group, pieces;
  bool edges;
};

// Rows stay in registers up to 512 threads with two pieces each, where the results begin on boundaries (`whole`: all rows of everything do).
static NormPlan norm_plan(int64_t width, int element, bool results, bool whole) {
  const int64_t pieces = width / (16 / element);
  NormPlan c{width <= 1024 ? 32 : 512, 0, false};
  if (!results || pieces == 0 || pieces > 1024) return c;
  c.edges = !whole;
  c.group = pieces <= 16 ? 16 : pieces <= 128 ? 32 : pieces <= 512 ? 128 : 512;
  c.pieces = c.group == 16 ? 1 : c.group == 32 ? (pieces <= 32 ? 1 : pieces <= 64 ? 2 : 4) : c.group == 128 ? (pieces <= 256 ? 2 : 4) : 2;
  return c;
}
static unsigned norm_blocks(const NormPlan& c, unsigned n, unsigned each) {
  const unsigned rows = (unsigned)(std::max(c.group, 128) / c.group);
  return std::min((n + rows - 1) / rows, each * (unsigned)plan_sm_count() / 8 * 8);      // (a group with several rows has them multiples of eight apart)
}
// Blocks of an SM in the gradient: two turns of those that it has at a time, which evens out that not all memory is as near to every SM,
// and few parts to add up.  (256 x 512 x 512 bf16, forward and backward with 8 and 5, 64 and 5, 64 and 10, 32 and 24 blocks an SM: 184, 206,
// 175, 190 us.)
static unsigned grad_blocks(const NormPlan& c, unsigned n) { return norm_blocks(c, n, c.group <= 128 ? 10 : 2); }
static unsigned grad_parts(const NormPlan& c, unsigned n) { return grad_blocks(c, n) * (c.pieces ? 1 : (unsigned)(std::max(c.group, 128) / c.group)); }

template <int P_, int G_>
struct NormCut {
  static constexpr int P = P_, G = G_, NT = G_ < 128 ? 128 : G_;
};
// f(NormCut<pieces, group>) of a plan.
template <typename F>
static int with_cut(const NormPlan& c, F&& f) {
  if (c.group == 16) return f(NormCut<1, 16>());
  if (c.group == 32) return c.pieces == 1 ? f(NormCut<1, 32>()) : c.pieces == 2 ? f(NormCut<2, 32>()) : f(NormCut<4, 32>());
  if (c.group == 128) return c.pieces == 2 ? f(NormCut<2, 128>()) : f(NormCut<4, 128>());
  return f(NormCut<2, 512>());
}

// Whether the rows of a strided tensor lie on the same addresses modulo 16 as those of a dense one that begins on 0.
static bool like_dense(const blstm_norm_desc& d, const void* p, const int64_t stride[2]) {
  const int64_t e = dtype_bytes(d.dtype);
  return p == nullptr || (aligned(16, p) && (d.n1 == 1 || ((stride[1] - d.width) * e & 15) == 0) && (d.n0 == 1 || ((stride[0] - d.n1 * d.width) * e & 15) == 0));
}

static bool whole_rows(const blstm_norm_desc& d, const void* weight) { return (d.width * dtype_bytes(d.dtype) & 15) == 0 && aligned(16, weight); }

static int check_norm(const blstm_norm_desc* d, const void* x, const void* weight) {
  if (!d || !valid_dtype(d->dtype) || !valid_rows(d->n0, d->n1) || d->width <= 0 || d->width > INT32_MAX / 2 || !(d->eps >= 0.f && d->eps < INFINITY))
    return BLSTM_E_INVALID_ARG;
  if (d->n0 && d->n1 && (!x || !weight || !aligned(dtype_bytes(d->dtype), x, weight))) return BLSTM_E_INVALID_ARG;
  return BLSTM_OK;
}

static NormParams norm_params(const blstm_norm_desc& d, const void* x, const void* r, const void* weight) {
  NormParams p{};
  p.x = x; p.r = r; p.w = weight;
  p.x_map = row_map(d.n0, d.n1, d.x_stride);
  p.r_map = row_map(d.n0, d.n1, d.residual_stride);
  p.dy_map = row_map(d.n0, d.n1, d.dy_stride);
  p.n = (unsigned)(d.n0 * d.n1); p.width = (unsigned)d.width;
  p.eps = d.eps;
  p.per_width = (float)(1.0 / (double)d.width);
  return p;
}

static int run_norm(const blstm_norm_desc& d, NormParams p, cudaStream_t st) {
  p.x_alike = like_dense(d, p.x, d.x_stride);
  p.r_alike = like_dense(d, p.r, d.residual_stride);
  const NormPlan c = norm_plan(d.width, dtype_bytes(d.dtype), aligned(16, p.y, p.h) && aligned(8, p.q), whole_rows(d, p.w) && p.x_alike && p.r_alike);
  const unsigned grid = norm_blocks(c, p.n, c.group <= 128 ? 64 : 4);
  return with_type(d.dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (c.pieces == 0) {
      if (c.group == 32) norm_any_kernel<T, 32><<<grid, 128, 0, st>>>(p);
      else norm_any_kernel<T, 512><<<grid, 512, 0, st>>>(p);
    } else {
      with_cut(c, [&](auto cut) -> int {
        using C = decltype(cut);
        if (c.edges) norm_kernel<T, C::P, C::G, true><<<grid, C::NT, 0, st>>>(p);
        else norm_kernel<T, C::P, C::G, false><<<grid, C::NT, 0, st>>>(p);
        return BLSTM_OK;
      });
    }
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    return BLSTM_OK;
  });
}

}  // namespace blstm

using namespace blstm;

extern "C" {

int blstm_rms_norm(const blstm_norm_desc* d, const void* x, const void* residual, const void* weight, void* y, void* sum, float* rstd, void* stream) {
  if (int rc = check_norm(d, x, weight)) return rc;
  if (d->n0 == 0 || d->n1 == 0) return BLSTM_OK;
  const size_t e = dtype_bytes(d->dtype);
  if (!y || !aligned(e, y, residual, sum) || (residual != nullptr) != (sum != nullptr) || !aligned(4, rstd)) return BLSTM_E_INVALID_ARG;
  NormParams p = norm_params(*d, x, residual, weight);
  p.y = y; p.h = sum; p.rstd = rstd;
  return run_norm(*d, p, (cudaStream_t)stream);
}

int blstm_rms_norm_e4m3(const blstm_norm_desc* d, const void* x, const void* residual, const void* weight, void* values, float* scales, void* sum,
                        void* stream) {
  if (int rc = check_norm(d, x, weight)) return rc;
  if (d->n0 == 0 || d->n1 == 0) return BLSTM_OK;
  const size_t e = dtype_bytes(d->dtype);
  if (!values || !scales || !aligned(4, scales) || !aligned(e, residual, sum) || (residual != nullptr) != (sum != nullptr)) return BLSTM_E_INVALID_ARG;
  NormParams p = norm_params(*d, x, residual, weight);
  p.q = static_cast<uint8_t*>(values); p.scales = scales; p.h = sum;
  return run_norm(*d, p, (cudaStream_t)stream);
}

// (the workspace of whichever cut has the more parts: where dx lies decides which one runs)
size_t blstm_rms_norm_grad_workspace(const blstm_norm_desc* d) {
  if (check_norm(d, reinterpret_cast<const void*>(16), reinterpret_cast<const void*>(16)) || d->n0 == 0 || d->n1 == 0) return 0;
  const unsigned n = (unsigned)(d->n0 * d->n1);
  unsigned parts = 1;
  for (const bool results : {false, true}) parts = std::max(parts, grad_parts(norm_plan(d->width, dtype_bytes(d->dtype), results, true), n));
  return round_up((size_t)parts * d->width * 4, 256);
}

int blstm_rms_norm_grad(const blstm_norm_desc* d, const void* dy, const void* dsum, const void* h, const void* weight, const float* rstd, void* dx,
                        void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_norm(d, h, weight)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const size_t e = dtype_bytes(d->dtype);
  if (!aligned(e, dy, dsum, dx, dweight) || !aligned(4, rstd)) return BLSTM_E_INVALID_ARG;
  if (d->n0 == 0 || d->n1 == 0) {
    if (dweight) BLSTM_CUDA_OK(cudaMemsetAsync(dweight, 0, d->width * e, st));
    return BLSTM_OK;
  }
  if (!dy || !rstd || !dx) return BLSTM_E_INVALID_ARG;
  if (dweight && (!workspace || !aligned(256, workspace) || workspace_bytes < blstm_rms_norm_grad_workspace(d))) return BLSTM_E_WORKSPACE;
  NormParams p = norm_params(*d, h, dsum, weight);
  p.dy = dy; p.y = dx;
  p.rstd = const_cast<float*>(rstd);
  p.x_alike = like_dense(*d, h, d->x_stride);
  p.r_alike = like_dense(*d, dsum, d->residual_stride);
  p.dy_alike = like_dense(*d, dy, d->dy_stride);
  const NormPlan c = norm_plan(d->width, (int)e, aligned(16, dx), whole_rows(*d, weight) && p.x_alike && p.r_alike && p.dy_alike);
  const unsigned grid = grad_blocks(c, p.n);
  p.parts = grad_parts(c, p.n);
  return with_type(d->dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (dweight) p.dw = static_cast<float*>(p.parts > 1 ? workspace : dweight);
    if (c.pieces == 0) {
      if (dweight) p.dw = static_cast<float*>(workspace);
      if (c.group == 32) norm_any_grad_kernel<T, 32><<<grid, 128, 0, st>>>(p);
      else norm_any_grad_kernel<T, 512><<<grid, 512, 0, st>>>(p);
    } else {
      with_cut(c, [&](auto cut) -> int {
        using C = decltype(cut);
        const size_t smem = (size_t)(C::NT / C::G) * (C::P * C::G + (c.edges ? 1 : 0)) * (kPer<T> + 1) * 4;
        static_assert((C::NT / C::G) * (C::P * C::G + 1) * (kPer<T> + 1) * 4 < 48 * 1024, "");
        if (c.edges) norm_grad_kernel<T, C::P, C::G, true><<<grid, C::NT, smem, st>>>(p);
        else norm_grad_kernel<T, C::P, C::G, false><<<grid, C::NT, smem, st>>>(p);
        return BLSTM_OK;
      });
    }
    BLSTM_CUDA_OK(cudaGetLastError());
    count_launch();
    if (dweight && (p.parts > 1 || c.pieces == 0)) {
      sum_parts_kernel<T><<<(p.width + 31) / 32, 32 * kSumWarps, 0, st>>>(static_cast<const float*>(workspace), static_cast<T*>(dweight), p.parts, p.width);
      BLSTM_CUDA_OK(cudaGetLastError());
      count_launch();
    }
    return BLSTM_OK;
  });
}

}  // extern "C"
