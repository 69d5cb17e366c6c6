// Layer normalisation over the rows of a matrix: forward, backward, and the backward of the backward pass.
//
// Row x of N values, mean() over the row (eps > 0):
//   forward      mu = mean(x), r = (mean((x - mu)^2) + eps)^-1/2, h = (x - mu) r, n = gamma h + beta, y = act(n)
//   backward     dn = act'(y) dy, g = gamma dn
//                dx = r (g - mean(g) - h mean(g h)), dgamma = sum_rows dn h, dbeta = sum_rows dn
//   second order (u: adjoint of dx)   q = r (u - mean(u) - h mean(u h))
//                ddy = act'(y) gamma q, dgamma = sum_rows dn q
//                dx = r^2 [h (3 mean(gh) mean(uh) + mean(g) mean(u) - mean(gu)) - mean(uh) (g - mean(g)) - mean(gh) (u - mean(u))]
//   (act is a leaky ReLU of slope >= 0, whose derivative follows from the sign of its output y)
//
// All three are bound by HBM: 8 to 30 flops per element of 2 to 6 arrays.  A row is read ONCE and kept in registers, as it
// was stored, by the G threads that own it (16, 64: part of or one wave, no barrier; 256, 1024: a workgroup), C vectors of
// 16 bytes each, so that the two passes of a centred variance and the 2 to 5 row means cost no second read.  Vectors are
// loaded at the element's alignment (the hardware needs no more), so odd widths and strides take the same path as padded
// ones; the up to 7 elements behind the last whole vector are one more element of as many threads.  From 4096 fp32 values on the
// backward passes read a row a second time where their registers do not suffice (back_holds), above 32768 all do.
// Measured (a copy of 1 GiB: 5.1 TB/s): forward 100000 x 256 33 us (6.2 TB/s, in part from the last-level cache), 4096 x 4297 bf16
// 16.6 us (4.2); backward with parameter gradients 40000 x 1000 bf16 66 us (4.8); second order 8192 x 1077 44 us (4.8).  Small
// calls are the host's: 32 x 256 11 us, of which the GPU works 3.4.
// Parameter gradients: every thread owns fixed columns, sums its rows in registers, the groups of a workgroup meet in
// LDS, and a second launch adds the workgroups' partial rows in a fixed order (no atomics: bit-reproducible).  A backward pass
// of few rows is one launch instead, with workgroups of columns beside those of rows: 1536 x 256 5.7 us of the GPU's instead of 7.6.
#include "agx_common.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int V = 4;
  typedef f32x4 __attribute__((aligned(4))) type;
};
template <> struct Vec<__bf16> {
  static constexpr int V = 8;
  typedef bf16x8 __attribute__((aligned(2))) type;
};

// A row as its group holds it: C whole vectors a thread, and one element of the row's end in the first few threads
template <typename T, int G, int C>
struct Row {
  static constexpr int V = Vec<T>::V;
  typename Vec<T>::type v[C];
  T end;
};
// where a thread's vectors and its end element are; the same for all rows of a launch
template <typename T, int G, int C>
struct Place {
  static constexpr int V = Vec<T>::V;
  int t, nv, last;               // thread of the group, whole vectors of a row, index of the end element or -1
  __device__ __forceinline__ explicit Place(int64_t n) : t(threadIdx.x % G), nv((int)(n / V)) {
    last = t < (int)(n - (int64_t)nv * V) ? nv * V + t : -1;
  }
  __device__ __forceinline__ bool in(int c) const { return c * G + t < nv; }
  __device__ __forceinline__ int at(int c) const { return (c * G + t) * V; }
  __device__ __forceinline__ typename Vec<T>::type vec(const T *p, int c) const {
    typename Vec<T>::type v = {};
    if (in(c)) v = *reinterpret_cast<const typename Vec<T>::type *>(p + at(c));
    return v;
  }
  __device__ __forceinline__ T end(const T *p) const { return last >= 0 ? p[last] : (T)0.f; }
  __device__ __forceinline__ void load(Row<T, G, C> &r, const T *__restrict__ p) const {
#pragma unroll
    for (int c = 0; c < C; ++c) r.v[c] = vec(p, c);
    r.end = end(p);
  }
};
// V parameters from p[i..]
template <int V>
__device__ __forceinline__ void load_param(const float *p, int i, float absent, float (&o)[V]) {
  if (!p) {
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] = absent;
    return;
  }
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const Vec<float>::type w = *reinterpret_cast<const Vec<float>::type *>(p + i + 4 * q);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[4 * q + k] = w[k];
  }
}
// parameters of a thread's columns, kept over all its rows where they are few
template <typename T, int G, int C>
struct Params {
  static constexpr int V = Vec<T>::V;
  static constexpr bool KEEP = C * V <= 16;
  const float *p;
  float absent, kept[KEEP ? C : 1][V], end;
  __device__ __forceinline__ Params(const float *p_, float absent_, const Place<T, G, C> &w) : p(p_), absent(absent_) {
    end = p && w.last >= 0 ? p[w.last] : absent;
    if constexpr (KEEP) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int k = 0; k < V; ++k) kept[c][k] = absent;
        if (w.in(c)) load_param<V>(p, w.at(c), absent, kept[c]);
      }
    }
  }
  __device__ __forceinline__ void get(const Place<T, G, C> &w, int c, float (&o)[V]) const {
    if constexpr (KEEP) {
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = kept[c][k];
    } else {
      load_param<V>(p, w.in(c) ? w.at(c) : 0, absent, o);
    }
  }
};

struct NormArgs {
  const void *x, *dy, *u, *ym;   // ym: forward output whose sign is the activation's derivative (NULL: no activation)
  void *y, *dx, *ddy;
  const float *gamma, *beta;
  float *mean, *rstd;
  const float *mean_in, *rstd_in;
  float *part;                   // [workgroups][2][width] partial parameter gradients (NULL: none wanted)
  int64_t ldx, lddy, ldu, ldym, ldy, lddx, ldddy;
  int64_t rows, n;
  float eps, slope;
  int act, add_dx;
};

// sums of K values over the G threads of a row's group; every thread gets them.  G > 64: `red` holds 2 * K * (G / 64)
// floats and `flip` alternates between its halves, so that one barrier a call is enough.
template <int G, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float *red, int &flip) {
#pragma unroll
  for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o, 64);
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    float *b = red + flip * K * W;
    flip ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) b[k * W + (threadIdx.x >> 6)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += b[k * W + w];
      v[k] = s;
    }
  }
}

template <int G> constexpr int block_threads() { return G > 256 ? G : 256; }

template <typename T, int G, int C>
__global__ __launch_bounds__(block_threads<G>()) void ln_fwd_kernel(NormArgs a) {
  constexpr int V = Vec<T>::V, NG = block_threads<G>() / G;
  __shared__ float red[G > 64 ? 2 * (G / 64) : 1];
  int flip = 0;
  const Place<T, G, C> w(a.n);
  const int grp = G == block_threads<G>() ? 0 : threadIdx.x / G;
  const float inv_n = 1.f / (float)a.n;
  const Params<T, G, C> gamma(a.gamma, 1.f, w), beta(a.beta, 0.f, w);
  auto act = [&](float n) { return a.act ? (n > 0.f ? n : a.slope * n) : n; };
  for (int64_t row = (int64_t)blockIdx.x * NG + grp; row < a.rows; row += (int64_t)gridDim.x * NG) {
    Row<T, G, C> x;
    w.load(x, reinterpret_cast<const T *>(a.x) + row * a.ldx);
    float s[1] = {(float)x.end};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) s[0] += (float)x.v[c][k];
    group_sum<G, 1>(s, red, flip);
    const float mu = s[0] * inv_n;
    const float de = (float)x.end - mu;
    s[0] = w.last >= 0 ? de * de : 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float q = 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = (float)x.v[c][k] - mu;
        q += d * d;
      }
      if (w.in(c)) s[0] += q;
    }
    group_sum<G, 1>(s, red, flip);
    const float r = 1.f / sqrtf(s[0] * inv_n + a.eps);
    if (w.t == 0) {
      if (a.mean) a.mean[row] = mu;
      if (a.rstd) a.rstd[row] = r;
    }
    T *y = reinterpret_cast<T *>(a.y) + row * a.ldy;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float ga[V], be[V];
      gamma.get(w, c, ga);
      beta.get(w, c, be);
      typename Vec<T>::type o;
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = (T)act(((float)x.v[c][k] - mu) * r * ga[k] + be[k]);
      if (w.in(c)) *reinterpret_cast<typename Vec<T>::type *>(y + w.at(c)) = o;
    }
    if (w.last >= 0) y[w.last] = (T)act(de * r * gamma.end + beta.end);
  }
}

// the workgroup's partial sums of NA parameter gradients: groups meet in LDS in a fixed order
template <typename T, int G, int C, int NA>
__device__ __forceinline__ void write_partials(float (&acc)[NA][C][Vec<T>::V], float (&end)[NA], const Place<T, G, C> &w,
                                               const NormArgs &a, float *lds) {
  constexpr int V = Vec<T>::V, NG = block_threads<G>() / G, W = G * C * V + V;   // (a group's columns, then its end elements)
  const int grp = G == block_threads<G>() ? 0 : threadIdx.x / G;
#pragma unroll
  for (int q = 0; q < NA; ++q) {
    float *p = a.part + ((int64_t)blockIdx.x * 2 + q) * a.n;
    if constexpr (NG > 1) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < V; ++k) lds[grp * W + w.at(c) + k] = acc[q][c][k];
      if (w.t < V) lds[grp * W + G * C * V + w.t] = end[q];
      __syncthreads();
      for (int i = threadIdx.x; i < a.n; i += block_threads<G>()) {
        const int o = i < w.nv * V ? i : G * C * V + i - w.nv * V;
        float s = 0.f;
        for (int g = 0; g < NG; ++g) s += lds[g * W + o];
        p[i] = s;
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (w.in(c))
#pragma unroll
          for (int k = 0; k < V; ++k) p[w.at(c) + k] = acc[q][c][k];
      if (w.last >= 0) p[w.last] = end[q];
    }
  }
}
template <typename T, int G, int C> constexpr int lds_floats() {
  return block_threads<G>() / G > 1 ? block_threads<G>() / G * (G * C * Vec<T>::V + Vec<T>::V) : 1;
}

// bit k of the result: the activation's derivative at element k is the slope (ym not positive)
template <typename T>
__device__ __forceinline__ uint32_t not_positive(const typename Vec<T>::type &m) {
  uint32_t b = 0;
#pragma unroll
  for (int k = 0; k < Vec<T>::V; ++k) b |= (float)m[k] > 0.f ? 0u : 1u << k;
  return b;
}

// One operand of the backward passes at a row.  HOLD: kept in registers; else each use reads it.
template <typename T, int G, int C, bool HOLD>
struct Operand {
  Row<T, G, C> held;
  const T *p;
  __device__ __forceinline__ void open(const Place<T, G, C> &w, const void *m, int64_t at) {
    p = reinterpret_cast<const T *>(m) + at;
    if constexpr (HOLD) w.load(held, p);
    else held.end = w.end(p);
  }
  __device__ __forceinline__ typename Vec<T>::type vec(const Place<T, G, C> &w, int c) const {
    if constexpr (HOLD) return held.v[c];
    else return w.vec(p, c);
  }
  __device__ __forceinline__ float end() const { return (float)held.end; }
};
// what the backward pass reads of a row
template <typename T, int G, int C, bool HOLD>
struct Inputs {
  Operand<T, G, C, HOLD> x, dy, m;
  float mu, r;
  __device__ __forceinline__ void load(const NormArgs &a, const Place<T, G, C> &w, int64_t row) {
    x.open(w, a.x, row * a.ldx);
    dy.open(w, a.dy, row * a.lddy);
    if (a.ym) m.open(w, a.ym, row * a.ldym);
    mu = a.mean_in[row];
    r = a.rstd_in[row];
  }
};
// (keeps a second reading of a row a reading, and how many vectors are in flight small)
__device__ __forceinline__ void read_again() { asm volatile("" ::: "memory"); }

// Rows of 1024 threads (8 to 32 values each, 128 registers a thread) are held where that leaves registers for the rest, else read
// again, from L2 or the last-level cache, which takes fewer.  Held and read again, us (the same inputs every pass): backward
// 2000 x 6000 (8 values) 38.1, 40.7; without sums 1000 x 14000 (16) 70, 77; with them 1800 x 9000 (12) 77, 68; second order
// 1000 x 6000 51, 35; 900 x 16000 179, 108; 1000 x 18154 bf16 206, 129.  What still spills, by hipcc's report: the second order
// with parameter gradients throughout (5 registers at 8 values to 69 at 32), without them up to 5, the backward pass with sums
// at 12 values 7 and without at 32 values 17.
constexpr bool back_holds(int g, int values, bool pg) { return g < 1024 || values <= (pg ? 8 : 16); }
constexpr bool back2_holds(int g) { return g < 1024; }
// the rows of workgroup `block` of `blocks`; lds: lds_floats<T, G, C>() where PG
template <typename T, int G, int C, bool PG>
__device__ __forceinline__ void back_rows(const NormArgs &a, int block, int blocks, float *lds) {
  constexpr int V = Vec<T>::V, NG = block_threads<G>() / G;
  __shared__ float red[G > 64 ? 2 * 2 * (G / 64) : 1];
  int flip = 0;
  const Place<T, G, C> w(a.n);
  const int grp = G == block_threads<G>() ? 0 : threadIdx.x / G;
  const float inv_n = 1.f / (float)a.n;
  const Params<T, G, C> gamma(a.gamma, 1.f, w);
  float acc[2][C][V] = {}, aend[2] = {0.f, 0.f};
  // (rows of one wave: the next one's loads are on their way while a row is worked on - 40000 x 1000 bf16 66 us instead of 68,
  //  20000 x 600 35 instead of 37 - where its registers do not cost a workgroup: 20000 x 2000 bf16 79 us without, 88 with)
  constexpr bool AHEAD = G <= 64 && C * V <= 16;
  const int64_t step = (int64_t)blocks * NG;
  int64_t row = (int64_t)block * NG + grp;
  constexpr bool HOLD = back_holds(G, C * V, PG);
  Inputs<T, G, C, HOLD> in;
  if (AHEAD && row < a.rows) in.load(a, w, row);
  for (; row < a.rows; row += step) {
    if (!AHEAD) in.load(a, w, row);
    const auto x = in.x, dy = in.dy;
    uint32_t neg[C] = {}, nend = 0;
    if (a.ym) {
#pragma unroll
      for (int c = 0; c < C; ++c) neg[c] = not_positive<T>(in.m.vec(w, c));
      nend = in.m.end() > 0.f ? 0u : 1u;
    }
    const float mu = in.mu, r = in.r;
    if (AHEAD && row + step < a.rows) in.load(a, w, row + step);
    auto hat = [&](float v) { return (v - mu) * r; };
    auto dn = [&](float v, int c, int k) { return neg[c] >> k & 1 ? a.slope * v : v; };
    const float he = w.last >= 0 ? hat(x.end()) : 0.f, de = nend ? a.slope * dy.end() : dy.end();
    const float ge = de * gamma.end;
    if constexpr (PG) {
      aend[0] += de * he;
      aend[1] += de;
    }
    float s[2] = {ge, ge * he};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float ga[V], q[2] = {0.f, 0.f};
      gamma.get(w, c, ga);
      if (!HOLD && c % 2 == 0) read_again();
      const auto xv = x.vec(w, c), dv = dy.vec(w, c);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float h = hat((float)xv[k]), d = dn((float)dv[k], c, k);
        if constexpr (PG) {
          acc[0][c][k] += d * h;
          acc[1][c][k] += d;
        }
        const float g = d * ga[k];
        q[0] += g;
        q[1] += g * h;
      }
      if (w.in(c)) {       // (behind the row's end d is 0, but h may not be finite)
        s[0] += q[0];
        s[1] += q[1];
      }
    }
    if (a.dx) {
      group_sum<G, 2>(s, red, flip);
        const float mg = s[0] * inv_n, mgh = s[1] * inv_n;
      T *dx = reinterpret_cast<T *>(a.dx) + row * a.lddx;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float ga[V];
        gamma.get(w, c, ga);
        if (!HOLD && c % 2 == 0) read_again();
      const auto xv = x.vec(w, c), dv = dy.vec(w, c);
        typename Vec<T>::type o = {};
        if (a.add_dx && w.in(c)) o = *reinterpret_cast<const typename Vec<T>::type *>(dx + w.at(c));
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = r * (dn((float)dv[k], c, k) * ga[k] - mg - hat((float)xv[k]) * mgh);
          o[k] = (T)(a.add_dx ? (float)o[k] + d : d);
        }
        if (w.in(c)) *reinterpret_cast<typename Vec<T>::type *>(dx + w.at(c)) = o;
      }
      if (w.last >= 0) {
        const float d = r * (ge - mg - he * mgh);
        dx[w.last] = (T)(a.add_dx ? (float)dx[w.last] + d : d);
      }
    }
  }
  if constexpr (PG) write_partials<T, G, C, 2>(acc, aend, w, a, lds);
}
template <typename T, int G, int C, bool PG>
__global__ __launch_bounds__(block_threads<G>()) void ln_bwd_kernel(NormArgs a) {
  __shared__ float lds[PG ? lds_floats<T, G, C>() : 1];
  back_rows<T, G, C, PG>(a, blockIdx.x, gridDim.x, lds);
}

// `left` of V values of a row; a row's terms of both parameter gradients
template <typename T>
__device__ __forceinline__ typename Vec<T>::type columns_at(const void *m, int64_t at, int left) {
  const T *p = reinterpret_cast<const T *>(m) + at;
  if (left == Vec<T>::V) return *reinterpret_cast<const typename Vec<T>::type *>(p);
  typename Vec<T>::type v = {};
#pragma unroll
  for (int k = 0; k < Vec<T>::V; ++k)
    if (k < left) v[k] = p[k];
  return v;
}
template <typename T>
__device__ __forceinline__ void add_columns(const NormArgs &a, const typename Vec<T>::type &x, const typename Vec<T>::type &dy, uint32_t neg,
                                            float mu, float r, float *dgamma, float *dbeta) {
#pragma unroll
  for (int k = 0; k < Vec<T>::V; ++k) {
    const float d = neg >> k & 1 ? a.slope * (float)dy[k] : (float)dy[k];
    dgamma[k] += d * (((float)x[k] - mu) * r);
    dbeta[k] += d;
  }
}

// Parameter gradients of V columns over all rows, by one workgroup of 256: with the statistics given they need no sum over a
// row.  A thread has every 256th row, U of them in flight (6: 512 x 256 4.1 us instead of 3.7); the threads meet in LDS in a
// fixed order.  Neighbouring strips are given to one XCD, which then fetches a line once for all of them: 1536 x 256 5.7 us, 12.8
// without.
template <typename T>
__device__ __forceinline__ void column_sums(const NormArgs &a, int strip, float *dgamma, float *dbeta, int accumulate, float *lds) {
  constexpr int V = Vec<T>::V, Q = 2 * V, LD = Q + 1, P = 256 / Q, U = 4;
  using VT = typename Vec<T>::type;
  const int64_t c0 = (int64_t)strip * V;
  const int left = (int)min((int64_t)V, a.n - c0);
  auto get = [&](const void *m, int64_t at) { return columns_at<T>(m, at + c0, left); };
  float s[Q] = {};
  for (int64_t row0 = threadIdx.x; row0 < a.rows; row0 += 256 * U) {
    VT x[U], dy[U], m[U];
    float mu[U], r[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t row = min(row0 + 256 * i, a.rows - 1);
      x[i] = get(a.x, row * a.ldx);
      dy[i] = get(a.dy, row * a.lddy);
      if (a.ym) m[i] = get(a.ym, row * a.ldym);
      mu[i] = a.mean_in[row];
      r[i] = a.rstd_in[row];
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (row0 + 256 * i < a.rows) add_columns<T>(a, x[i], dy[i], a.ym ? not_positive<T>(m[i]) : 0u, mu[i], r[i], s, s + V);
  }
  const int t = threadIdx.x, q = t % Q, part = t / Q;
#pragma unroll
  for (int k = 0; k < Q; ++k) lds[t * LD + k] = s[k];
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < Q; ++i) sum += lds[(part * Q + i) * LD + q];
  __syncthreads();
  lds[part * LD + q] = sum;
  __syncthreads();
  float *out = q < V ? dgamma : dbeta;
  if (part == 0 && out && q % V < left) {
    out += c0 + q % V;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) sum += lds[i * LD + q];
    *out = accumulate ? *out + sum : sum;              // (what is there is added last: one rounding against it)
  }
}
template <typename T> constexpr int strip_floats() { return 256 * (2 * Vec<T>::V + 1); }
// the whole backward pass in one launch: the first `strips` workgroups are columns', the others rows'
template <typename T, int G, int C>
__global__ __launch_bounds__(256) void ln_bwd_small_kernel(NormArgs a, int strips, float *dgamma, float *dbeta, int accumulate) {
  __shared__ float lds[strip_floats<T>()];
  if ((int)blockIdx.x < strips) column_sums<T>(a, agx::xcd_logical_id(blockIdx.x, strips), dgamma, dbeta, accumulate, lds);
  else back_rows<T, G, C, false>(a, blockIdx.x - strips, gridDim.x - strips, lds);
}

template <typename T, int G, int C, bool PG>
__global__ __launch_bounds__(block_threads<G>()) void ln_bwd2_kernel(NormArgs a) {
  constexpr int V = Vec<T>::V, NG = block_threads<G>() / G;
  __shared__ float red[G > 64 ? 2 * 5 * (G / 64) : 1];
  __shared__ float lds[PG ? lds_floats<T, G, C>() : 1];
  constexpr bool HOLD = back2_holds(G);
  int flip = 0;
  const Place<T, G, C> w(a.n);
  const int grp = G == block_threads<G>() ? 0 : threadIdx.x / G;
  const float inv_n = 1.f / (float)a.n;
  const Params<T, G, C> gamma(a.gamma, 1.f, w);
  float acc[1][C][V] = {}, aend[1] = {0.f};
  for (int64_t row = (int64_t)blockIdx.x * NG + grp; row < a.rows; row += (int64_t)gridDim.x * NG) {
    Operand<T, G, C, HOLD> x, dy, u;
    uint32_t neg[C] = {}, nend = 0;
    x.open(w, a.x, row * a.ldx);
    dy.open(w, a.dy, row * a.lddy);
    u.open(w, a.u, row * a.ldu);
    if (a.ym) {
      Operand<T, G, C, HOLD> m;
      m.open(w, a.ym, row * a.ldym);
#pragma unroll
      for (int c = 0; c < C; ++c) neg[c] = not_positive<T>(m.vec(w, c));
      nend = m.end() > 0.f ? 0u : 1u;
    }
    const float mu = a.mean_in[row], r = a.rstd_in[row];
    auto hat = [&](float v) { return (v - mu) * r; };
    auto dn = [&](float v, int c, int k) { return neg[c] >> k & 1 ? a.slope * v : v; };
    const float he = w.last >= 0 ? hat(x.end()) : 0.f, de = nend ? a.slope * dy.end() : dy.end();
    const float ge = de * gamma.end, ue = u.end();
    float s[5] = {ge, ge * he, ue, ue * he, ge * ue};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float ga[V], q[5] = {};
      gamma.get(w, c, ga);
      if (!HOLD && c % 2 == 0) read_again();
      const auto xv = x.vec(w, c), dv = dy.vec(w, c), uv = u.vec(w, c);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float h = hat((float)xv[k]), g = dn((float)dv[k], c, k) * ga[k], uu = (float)uv[k];
        q[0] += g;
        q[1] += g * h;
        q[2] += uu;
        q[3] += uu * h;
        q[4] += g * uu;
      }
      if (w.in(c))
#pragma unroll
        for (int k = 0; k < 5; ++k) s[k] += q[k];
    }
    group_sum<G, 5>(s, red, flip);
    const float mg = s[0] * inv_n, mgh = s[1] * inv_n, mu_ = s[2] * inv_n, muh = s[3] * inv_n, mgu = s[4] * inv_n;
    const float hc = 3.f * mgh * muh + mg * mu_ - mgu, r2 = r * r;
    T *dx = reinterpret_cast<T *>(a.dx) + row * a.lddx;
    T *ddy = reinterpret_cast<T *>(a.ddy) + row * a.ldddy;
    auto second = [&](float h, float g, float uu) { return r2 * (h * hc - muh * (g - mg) - mgh * (uu - mu_)); };
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float ga[V];
      gamma.get(w, c, ga);
      if (!HOLD && c % 2 == 0) read_again();
      const auto xv = x.vec(w, c), dv = dy.vec(w, c), uv = u.vec(w, c);
      typename Vec<T>::type o = {}, e;
      if (a.dx && a.add_dx && w.in(c)) o = *reinterpret_cast<const typename Vec<T>::type *>(dx + w.at(c));
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float h = hat((float)xv[k]), d = dn((float)dv[k], c, k), uu = (float)uv[k];
        const float q = r * (uu - mu_ - h * muh);
        if constexpr (PG) acc[0][c][k] += d * q;
        e[k] = (T)(neg[c] >> k & 1 ? ga[k] * q * a.slope : ga[k] * q);
        const float b = second(h, d * ga[k], uu);
        o[k] = (T)(a.add_dx ? (float)o[k] + b : b);
      }
      if (a.dx && w.in(c)) *reinterpret_cast<typename Vec<T>::type *>(dx + w.at(c)) = o;
      if (a.ddy && w.in(c)) *reinterpret_cast<typename Vec<T>::type *>(ddy + w.at(c)) = e;
    }
    if (w.last >= 0) {
      const float q = r * (ue - mu_ - he * muh), b = second(he, ge, ue);
      if constexpr (PG) aend[0] += de * q;
      if (a.dx) dx[w.last] = (T)(a.add_dx ? (float)dx[w.last] + b : b);
      if (a.ddy) ddy[w.last] = (T)(nend ? gamma.end * q * a.slope : gamma.end * q);
    }
  }
  if constexpr (PG) write_partials<T, G, C, 1>(acc, aend, w, a, lds);
}

// Rows of more than 32768 values: one workgroup a row, the row read again for each pass (it stays in L2 between them).  The second
// order's partial parameter gradients are added to the workgroup's own row of `part`, each column by one thread; the backward
// pass has them apart (ln_columns_kernel).
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(NormArgs a) {
  __shared__ float red[2 * 16];
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = reinterpret_cast<const T *>(a.x) + row * a.ldx;
    float s[1] = {0.f};
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) s[0] += (float)x[i];
    group_sum<1024, 1>(s, red, flip);
    const float mu = s[0] / (float)a.n;
    s[0] = 0.f;
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
      const float d = (float)x[i] - mu;
      s[0] += d * d;
    }
    group_sum<1024, 1>(s, red, flip);
    const float r = 1.f / sqrtf(s[0] / (float)a.n + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mu;
      if (a.rstd) a.rstd[row] = r;
    }
    T *y = reinterpret_cast<T *>(a.y) + row * a.ldy;
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
      const float n = ((float)x[i] - mu) * r * (a.gamma ? a.gamma[i] : 1.f) + (a.beta ? a.beta[i] : 0.f);
      y[i] = (T)(a.act ? (n > 0.f ? n : a.slope * n) : n);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_wide_kernel(NormArgs a) {
  __shared__ float red[2 * 2 * 16];
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = reinterpret_cast<const T *>(a.x) + row * a.ldx;
    const T *dy = reinterpret_cast<const T *>(a.dy) + row * a.lddy;
    const T *ym = a.ym ? reinterpret_cast<const T *>(a.ym) + row * a.ldym : nullptr;
    const float mu = a.mean_in[row], r = a.rstd_in[row];
    float s[2] = {0.f, 0.f};
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
      float d = (float)dy[i];
      if (ym && !((float)ym[i] > 0.f)) d *= a.slope;
      const float h = ((float)x[i] - mu) * r;
      const float g = d * (a.gamma ? a.gamma[i] : 1.f);
      s[0] += g;
      s[1] += g * h;
    }
    group_sum<1024, 2>(s, red, flip);
    const float mg = s[0] / (float)a.n, mgh = s[1] / (float)a.n;
    T *dx = reinterpret_cast<T *>(a.dx) + row * a.lddx;
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
      float d = (float)dy[i];
      if (ym && !((float)ym[i] > 0.f)) d *= a.slope;
      const float h = ((float)x[i] - mu) * r;
      const float o = r * (d * (a.gamma ? a.gamma[i] : 1.f) - mg - h * mgh);
      dx[i] = (T)(a.add_dx ? (float)dx[i] + o : o);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd2_wide_kernel(NormArgs a) {
  __shared__ float red[2 * 5 * 16];
  int flip = 0;
  float *p0 = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.n : nullptr;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = reinterpret_cast<const T *>(a.x) + row * a.ldx;
    const T *dy = reinterpret_cast<const T *>(a.dy) + row * a.lddy;
    const T *up = reinterpret_cast<const T *>(a.u) + row * a.ldu;
    const T *ym = a.ym ? reinterpret_cast<const T *>(a.ym) + row * a.ldym : nullptr;
    const float mu = a.mean_in[row], r = a.rstd_in[row];
    float s[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
      float d = (float)dy[i];
      if (ym && !((float)ym[i] > 0.f)) d *= a.slope;
      const float h = ((float)x[i] - mu) * r, g = d * (a.gamma ? a.gamma[i] : 1.f), u = (float)up[i];
      s[0] += g;
      s[1] += g * h;
      s[2] += u;
      s[3] += u * h;
      s[4] += g * u;
    }
    group_sum<1024, 5>(s, red, flip);
    const float n = (float)a.n, mg = s[0] / n, mgh = s[1] / n, mu_ = s[2] / n, muh = s[3] / n, mgu = s[4] / n;
    const float hc = 3.f * mgh * muh + mg * mu_ - mgu, r2 = r * r;
    T *dx = reinterpret_cast<T *>(a.dx) + row * a.lddx;
    T *ddy = reinterpret_cast<T *>(a.ddy) + row * a.ldddy;
    for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
      const bool neg = ym && !((float)ym[i] > 0.f);
      const float d = neg ? (float)dy[i] * a.slope : (float)dy[i];
      const float ga = a.gamma ? a.gamma[i] : 1.f, h = ((float)x[i] - mu) * r, u = (float)up[i];
      const float q = r * (u - mu_ - h * muh);
      if (p0) p0[i] = (first ? 0.f : p0[i]) + d * q;
      if (a.dx) {
        const float b = r2 * (h * hc - muh * (d * ga - mg) - mgh * (u - mu_));
        dx[i] = (T)(a.add_dx ? (float)dx[i] + b : b);
      }
      if (a.ddy) ddy[i] = (T)(neg ? ga * q * a.slope : ga * q);
    }
    first = false;
  }
}

// Parameter gradients of the backward pass by itself, for rows whose workgroup has no registers for them: a thread has V columns
// and every gridDim.y-th row; partial sums as above.
template <typename T>
__global__ __launch_bounds__(256) void ln_columns_kernel(NormArgs a) {
  constexpr int V = Vec<T>::V, U = 4;
  const int64_t c0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (c0 >= a.n) return;
  const int left = (int)min((int64_t)V, a.n - c0);
  float s[2][V] = {};
  const int64_t step = gridDim.y;
  for (int64_t row0 = blockIdx.y; row0 < a.rows; row0 += U * step) {
    typename Vec<T>::type x[U], dy[U], m[U];
    float mu[U], r[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t row = min(row0 + i * step, a.rows - 1);
      x[i] = columns_at<T>(a.x, row * a.ldx + c0, left);
      dy[i] = columns_at<T>(a.dy, row * a.lddy + c0, left);
      if (a.ym) m[i] = columns_at<T>(a.ym, row * a.ldym + c0, left);
      mu[i] = a.mean_in[row];
      r[i] = a.rstd_in[row];
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (row0 + i * step < a.rows) add_columns<T>(a, x[i], dy[i], a.ym ? not_positive<T>(m[i]) : 0u, mu[i], r[i], s[0], s[1]);
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float *p = a.part + ((int64_t)blockIdx.y * 2 + q) * a.n + c0;
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) p[k] = s[q][k];
  }
}

// out_q[j] (+)= sum over workgroups b of part[b][q][j], b in a fixed order: 32 columns by 32 interleaved shares a workgroup, which
// takes every gridDim.x-th such piece (a launch has fewer than 2^32 threads along x: 2^27 columns at a piece a workgroup)
constexpr int MAX_PIECES = 1 << 20;
__global__ __launch_bounds__(1024) void ln_param_kernel(const float *__restrict__ part, int nb, int64_t n, float *dgamma,
                                                        float *dbeta, int accumulate) {
  __shared__ float red[32][33];
  float *out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  const int col = threadIdx.x & 31, sh = threadIdx.x >> 5;
  for (int64_t j0 = (int64_t)blockIdx.x * 32; j0 < n; j0 += (int64_t)gridDim.x * 32) {
    const int64_t j = j0 + col;
    float s = 0.f;
    if (j < n) {
#pragma unroll 8
      for (int b = sh; b < nb; b += 32) s += part[((int64_t)b * 2 + blockIdx.y) * n + j];
    }
    red[sh][col] = s;
    __syncthreads();
    if (sh == 0 && j < n) {
      s = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) s += red[k][col];
      out[j] = accumulate ? out[j] + s : s;
    }
    __syncthreads();
  }
}

enum { FWD, BWD, BWD2 };
constexpr int PARAM_BLOCKS = 4;

// One round of workgroups, as many as the kernel's registers let a CU hold: a second round would leave most of it idle, and a
// workgroup more or less a CU is worth a lot (backward, a CU 2, 3, 4 and 6 of them: 40000 x 1000 bf16, of which 3 fit, 67, 67,
// 78, 73 us; 6000 x 4297 bf16, 2 fit, 68, 88, 76, 90; second order of 8192 x 1077, 4 fit, 55, 45, 44, 49).
template <auto KERNEL> int resident(int threads) {
  static const int n = [&] {
    int fit = 0;
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(&fit, KERNEL, threads, 0) == hipSuccess ? std::max(1, fit) : 1;
  }();
  return n;
}
template <auto KERNEL> void launch_one(hipStream_t st, const NormArgs &a, int threads, int &blocks) {
  blocks = std::min(blocks, agx::num_cus() * resident<KERNEL>(threads));
  hipLaunchKernelGGL(KERNEL, dim3(blocks), dim3(threads), 0, st, a);
}
// rows whose workgroup sums no parameter gradients in the backward pass (g: 0, or the threads of a row, values of each):
// their sums take another launch (ln_columns_kernel), which reads x, dy and y once more.  Values, us in the rows' workgroups and
// apart: 12 (1800 x 9000) 68, 80; 16 (1000 x 14000) 96, 70; 20 (800 x 18154) 119, 90; 24 (2000 x 18154 bf16) 246, 139.
constexpr bool params_apart(int g, int values) { return g == 0 || (g == 1024 && values > 12); }

template <int OP, typename T, int G, int C>
void launch_cfg(hipStream_t st, const NormArgs &a, int &blocks) {
  constexpr int threads = block_threads<G>();
  if constexpr (OP == FWD) launch_one<&ln_fwd_kernel<T, G, C>>(st, a, threads, blocks);
  else if constexpr (OP == BWD) {
    if constexpr (!params_apart(G, C * Vec<T>::V))
      if (a.part) return launch_one<&ln_bwd_kernel<T, G, C, true>>(st, a, threads, blocks);
    launch_one<&ln_bwd_kernel<T, G, C, false>>(st, a, threads, blocks);
  } else {
    if (a.part) launch_one<&ln_bwd2_kernel<T, G, C, true>>(st, a, threads, blocks);
    else launch_one<&ln_bwd2_kernel<T, G, C, false>>(st, a, threads, blocks);
  }
}

// threads a row's group has (0: the wide kernels) and vectors each of them holds, by the row's whole vectors of 16 bytes
struct Cfg { int g, c; };
Cfg pick(int64_t width, int v) {
  const int64_t nv = std::max<int64_t>(1, width / v);
  if (nv <= 16) return {16, 1};
  if (nv <= 64 * 4) return {64, (int)agx::cdiv64(nv, 64)};
  if (nv <= 256 * 4) return {256, (int)agx::cdiv64(nv, 256)};
  if (nv <= 1024 * (32 / v)) return {1024, (int)agx::cdiv64(nv, 1024)};
  return {0, 0};
}
// workgroups of a launch at most: a row each; with parameter gradients PARAM_BLOCKS a CU, because each writes and the second
// launch reads a partial row (the workspace is made for these)
int blocks_of(int64_t rows, const Cfg &c, bool params) {
  const int ng = c.g == 0 || c.g >= 256 ? 1 : 256 / c.g;
  return (int)std::min<int64_t>(agx::cdiv64(rows, ng), (int64_t)agx::num_cus() * (params ? PARAM_BLOCKS : 16));
}

// calls f with a configuration's G and C as constants; false: the wide kernels' rows
template <int V, class F> bool by_cfg(const Cfg &c, F f) {
  auto by_c = [&](auto g) {
    if constexpr (decltype(g)::value == 64)                             // (wider groups have more: see pick)
      if (c.c == 1) return f(g, std::integral_constant<int, 1>{});
    if (c.c == 2) f(g, std::integral_constant<int, 2>{});
    else if (c.c == 3) f(g, std::integral_constant<int, 3>{});
    else if (c.c == 4) f(g, std::integral_constant<int, 4>{});
    else if constexpr (decltype(g)::value == 1024 && V == 4) {
      if (c.c == 5) f(g, std::integral_constant<int, 5>{});
      else if (c.c == 6) f(g, std::integral_constant<int, 6>{});
      else f(g, std::integral_constant<int, 8>{});
    }
  };
  if (c.g == 16) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  else if (c.g == 64) by_c(std::integral_constant<int, 64>{});
  else if (c.g == 256) by_c(std::integral_constant<int, 256>{});
  else if (c.g == 1024) by_c(std::integral_constant<int, 1024>{});
  return c.g != 0;
}

// The backward pass with parameter gradients in one launch (ln_bwd_small_kernel) instead of two, up to SMALL_ROWS rows - six a
// thread of a columns' workgroup, up to which it is no slower at any width - and SMALL_VECTORS whole vectors a matrix.  GPU time of
// two launches and one, us: 16 x 256 5.1, 3.2; widths 64, 256, 512, 1024 by 512 rows 5.4, 3.6; 6.5, 3.7; 7.3, 4.0; 8.9, 5.9;
// by 1024 5.8, 4.0; 6.3, 4.4; 7.2, 5.6; 9.4, 8.0; by 1536 6.0, 5.3; 7.6, 5.7; 8.9, 6.8; 11.6, 11.4 (bf16 6.4, 5.9; 8.1, 6.3; 8.4,
// 6.5; 10.9, 7.7); by 2048 6.4, 5.7; 7.5, 6.7; 9.0, 7.9; 12.7, 15.5 (bf16 6.7, 6.7; 7.8, 7.2; 8.3, 7.7; 11.1, 9.0); by 3000 6.9,
// 7.5; 9.8, 8.6; 11.8, 16.4; 16.6, 20.3; by 4096 6.0, 9.2; 10.2, 10.5; 13.1, 22.0; 19.0, 25.2.  2048 x 600 9.9, 11.7; 512 x 4000
// 16.0, 14.8; 1024 x 4000 21.4, 25.4; 512 x 4297 bf16 22.5, 13.1.  (The host's second launch costs 3.4 us more.)
constexpr int SMALL_ROWS = 1536, SMALL_VECTORS = 1 << 19;
bool small_shape(int64_t rows, int64_t width, int v) {
  const int g = pick(width, v).g;
  return rows > 0 && rows <= SMALL_ROWS && rows * (width / v) <= SMALL_VECTORS && g != 0 && g <= 256;
}
bool small_back(const NormArgs &a, const float *dgamma, const float *dbeta, int v) {
  // (not where dx is written over what the columns' workgroups still read)
  const bool over = a.dx && (a.dx == a.x || a.dx == a.dy || a.dx == a.ym);
  return (dgamma || dbeta) && !over && small_shape(a.rows, a.n, v);
}

template <int OP, typename T>
int launch(hipStream_t st, const NormArgs &a, float *dgamma, float *dbeta, int accumulate) {
  const Cfg c = pick(a.n, Vec<T>::V);
  if constexpr (OP == BWD)
    if (small_back(a, dgamma, dbeta, Vec<T>::V)) {
      const int strips = (int)agx::cdiv64(a.n, Vec<T>::V), rows = a.dx ? blocks_of(a.rows, c, false) : 0;
      by_cfg<Vec<T>::V>(c, [&](auto g, auto n) {
        if constexpr (decltype(g)::value <= 256)
          hipLaunchKernelGGL((ln_bwd_small_kernel<T, decltype(g)::value, decltype(n)::value>), dim3(strips + rows), dim3(256), 0, st, a,
                             strips, dgamma, dbeta, accumulate);
      });
      AGX_LAUNCH_CHECK();
      return AGX_OK;
    }
  NormArgs rows = a;
  int blocks = blocks_of(a.rows, c, a.part != nullptr), parts = 0;
  if constexpr (OP == BWD)
    if (a.part && a.rows > 0 && params_apart(c.g, c.c * Vec<T>::V)) {          // (before the rows: dx may be written over an input)
      const int cols = (int)agx::cdiv64(a.n, 256 * Vec<T>::V);
      parts = (int)std::min<int64_t>(a.rows, std::max(1, agx::num_cus() * PARAM_BLOCKS / cols));
      hipLaunchKernelGGL(ln_columns_kernel<T>, dim3(cols, parts), dim3(256), 0, st, a);
      AGX_LAUNCH_CHECK();
      rows.part = nullptr;
      blocks = a.dx ? blocks_of(a.rows, c, false) : 0;
    }
  if (blocks > 0) {
    if (!by_cfg<Vec<T>::V>(c, [&](auto g, auto n) { launch_cfg<OP, T, decltype(g)::value, decltype(n)::value>(st, rows, blocks); })) {
      if constexpr (OP == FWD) launch_one<&ln_fwd_wide_kernel<T>>(st, rows, 1024, blocks);
      else if constexpr (OP == BWD) launch_one<&ln_bwd_wide_kernel<T>>(st, rows, 1024, blocks);
      else launch_one<&ln_bwd2_wide_kernel<T>>(st, rows, 1024, blocks);
    }
    AGX_LAUNCH_CHECK();
  }
  if (dgamma || dbeta) {
    hipLaunchKernelGGL(ln_param_kernel, dim3((unsigned)std::min<int64_t>(agx::cdiv64(a.n, 32), MAX_PIECES), 2), dim3(1024), 0, st, a.part,
                       parts ? parts : blocks, a.n, dgamma, dbeta, accumulate);
    AGX_LAUNCH_CHECK();
  }
  return AGX_OK;
}

int vector_of(int32_t dtype) { return dtype == AGX_BF16 ? 8 : 4; }
int check_norm(const agx_norm_t *p, const char *who) {
  AGX_CHECK_ARG(p, "%s: null argument", who);
  AGX_CHECK_ARG(p->dtype == AGX_F32 || p->dtype == AGX_BF16, "%s: dtype %d", who, p->dtype);
  AGX_CHECK_ARG(p->rows >= 0 && p->width > 0 && p->width <= (1 << 28), "%s: rows %lld, width %lld", who, (long long)p->rows,
                (long long)p->width);
  AGX_CHECK_ARG(p->slope >= 0.f && p->slope <= 1.f, "%s: slope must be in [0, 1]", who);
  AGX_CHECK_ARG(p->act == 0 || p->act == 1, "%s: act %d", who, p->act);
  return AGX_OK;
}
int check_mat(const agx_norm_t *p, const void *m, int64_t ld, const char *who, const char *name) {
  AGX_CHECK_ARG(m && ld >= p->width, "%s: %s missing or its leading dimension below the width", who, name);
  const uintptr_t al = p->dtype == AGX_F32 ? 3 : 1;
  AGX_CHECK_ARG((reinterpret_cast<uintptr_t>(m) & al) == 0, "%s: %s not aligned to its elements", who, name);
  return AGX_OK;
}
NormArgs back_args(const agx_norm_t *p) {
  NormArgs a = {};
  a.x = p->x; a.dy = p->dy; a.ym = p->act ? p->y : nullptr; a.dx = p->dx;
  a.ldx = p->ldx; a.lddy = p->lddy; a.ldym = p->act ? p->ldy : 0; a.lddx = p->lddx;
  a.gamma = p->gamma; a.mean_in = p->mean; a.rstd_in = p->rstd;
  a.part = (p->dgamma || p->dbeta) ? p->ws : nullptr;
  a.rows = p->rows; a.n = p->width; a.slope = p->slope; a.act = p->act; a.add_dx = p->accumulate_dx ? 1 : 0;
  return a;
}
// What a call writes shares no element with anything else of its descriptor, but that an output may be the same matrix as an
// input (a thread has read a place of it before it writes there).
int check_overlaps(const agx_norm_t *p, int op, const char *who) {
  const int bytes = p->dtype == AGX_F32 ? 4 : 2;
  const bool back = op != FWD, params = p->dgamma || p->dbeta;
  auto matrix = [&](const void *m, int64_t ld) { return agx::Region{m, p->rows, p->width, ld, bytes}; };
  auto vec = [](const float *v, int64_t n) { return agx::Region{n > 0 ? v : nullptr, 1, n, n, 4}; };
  struct Vector { agx::Region r; const char *name, *written; };                  // written: what it is where the call writes it
  const char *stat = back ? nullptr : "a statistic", *grad = back ? "a parameter gradient" : nullptr;
  const Vector vectors[7] = {
      {vec(p->gamma, p->width), "gamma", nullptr}, {vec(p->beta, p->width), "beta", nullptr},
      {vec(p->mean, p->rows), "mean", stat}, {vec(p->rstd, p->rows), "rstd", stat},
      {vec(p->dgamma, p->width), "dgamma", grad}, {vec(p->dbeta, p->width), "dbeta", grad},
      {vec(params ? p->ws : nullptr, std::min(p->ws_floats, agx_layernorm_ws_floats(p->rows, p->width, p->dtype))), "the workspace",
       back ? "the workspace" : nullptr}};
  struct Matrix { agx::Region r; const char *name; };
  const Matrix in[4] = {{matrix(p->x, p->ldx), "x"},
                        {matrix(back ? p->dy : nullptr, p->lddy), "dy"},
                        {matrix(op == BWD2 ? p->u : nullptr, p->ldu), "u"},
                        {matrix(back && p->act ? p->y : nullptr, p->ldy), "y"}};
  const agx::Region out[2] = {back ? matrix(p->dx, p->lddx) : matrix(p->y, p->ldy), matrix(op == BWD2 ? p->ddy : nullptr, p->ldddy)};
  for (int i = 0; i < 7; ++i)
    for (int k = 0; k < 7; ++k)
      AGX_CHECK_ARG(k == i || !vectors[i].written || !agx::overlap(vectors[i].r, vectors[k].r),
                    "%s: %s overlaps %s", who, vectors[i].written, vectors[k].name);
  for (const Vector &v : vectors) {
    for (const Matrix &m : in)
      AGX_CHECK_ARG(!v.written || !agx::overlap(v.r, m.r), "%s: %s overlaps %s", who, v.written, m.name);
    for (const agx::Region &o : out) AGX_CHECK_ARG(!agx::overlap(o, v.r), "%s: an output matrix overlaps %s", who, v.name);
  }
  for (const agx::Region &o : out)
    for (const Matrix &m : in)
      AGX_CHECK_ARG((o.p == m.r.p && (o.ld == m.r.ld || p->rows == 1)) || !agx::overlap(o, m.r),
                    "%s: an output matrix overlaps %s without being the same matrix", who, m.name);
  AGX_CHECK_ARG(!agx::overlap(out[0], out[1]), "%s: dx and ddy overlap", who);
  return AGX_OK;
}
int check_back(const agx_norm_t *p, bool second, const char *who) {
  AGX_TRY(check_mat(p, p->x, p->ldx, who, "x"));
  AGX_TRY(check_mat(p, p->dy, p->lddy, who, "dy"));
  AGX_CHECK_ARG(p->mean && p->rstd, "%s: mean / rstd missing", who);
  if (p->act) AGX_TRY(check_mat(p, p->y, p->ldy, who, "y"));
  if (p->dx) AGX_TRY(check_mat(p, p->dx, p->lddx, who, "dx"));
  if (second) {
    AGX_TRY(check_mat(p, p->u, p->ldu, who, "u"));
    if (p->ddy) AGX_TRY(check_mat(p, p->ddy, p->ldddy, who, "ddy"));
  }
  if (p->dgamma || p->dbeta) {
    const int64_t need = !second && small_back(back_args(p), p->dgamma, p->dbeta, vector_of(p->dtype))
                             ? 0
                             : agx_layernorm_ws_floats(p->rows, p->width, p->dtype);
    if (need > 0 && (!p->ws || p->ws_floats < need)) {
      agx::set_error("%s: workspace of %lld floats, %lld needed", who, (long long)p->ws_floats, (long long)need);
      return AGX_E_WORKSPACE;
    }
  }
  return check_overlaps(p, second ? BWD2 : BWD, who);
}

}  // namespace

extern "C" int64_t agx_layernorm_ws_floats(int64_t rows, int64_t width, int32_t dtype) {
  if (rows <= 0 || width <= 0) return 0;
  return (int64_t)blocks_of(rows, pick(width, vector_of(dtype)), true) * 2 * width;
}

extern "C" int64_t agx_layernorm_bwd_ws_floats(int64_t rows, int64_t width, int32_t dtype) {
  return rows > 0 && width > 0 && small_shape(rows, width, vector_of(dtype)) ? 0 : agx_layernorm_ws_floats(rows, width, dtype);
}

extern "C" int agx_layernorm_fwd(void *stream, const agx_norm_t *p) {
  AGX_TRY(check_norm(p, "agx_layernorm_fwd"));
  AGX_CHECK_ARG(p->eps > 0.f, "agx_layernorm_fwd: eps must be positive");
  if (p->rows == 0) return AGX_OK;
  AGX_TRY(check_mat(p, p->x, p->ldx, "agx_layernorm_fwd", "x"));
  AGX_TRY(check_mat(p, p->y, p->ldy, "agx_layernorm_fwd", "y"));
  AGX_TRY(check_overlaps(p, FWD, "agx_layernorm_fwd"));
  NormArgs a = {};
  a.x = p->x; a.ldx = p->ldx; a.y = p->y; a.ldy = p->ldy;
  a.gamma = p->gamma; a.beta = p->beta; a.mean = p->mean; a.rstd = p->rstd;
  a.rows = p->rows; a.n = p->width; a.eps = p->eps; a.slope = p->slope; a.act = p->act;
  return p->dtype == AGX_F32 ? launch<FWD, float>(agx::as_stream(stream), a, nullptr, nullptr, 0)
                             : launch<FWD, __bf16>(agx::as_stream(stream), a, nullptr, nullptr, 0);
}

extern "C" int agx_layernorm_bwd(void *stream, const agx_norm_t *p) {
  AGX_TRY(check_norm(p, "agx_layernorm_bwd"));
  if (p->rows > 0) AGX_TRY(check_back(p, false, "agx_layernorm_bwd"));
  AGX_CHECK_ARG(p->dx || p->dgamma || p->dbeta || p->rows == 0, "agx_layernorm_bwd: no output wanted");
  const NormArgs a = back_args(p);
  return p->dtype == AGX_F32
             ? launch<BWD, float>(agx::as_stream(stream), a, p->dgamma, p->dbeta, p->accumulate_params)
             : launch<BWD, __bf16>(agx::as_stream(stream), a, p->dgamma, p->dbeta, p->accumulate_params);
}

extern "C" int agx_layernorm_bwd2(void *stream, const agx_norm_t *p) {
  AGX_TRY(check_norm(p, "agx_layernorm_bwd2"));
  AGX_CHECK_ARG(!p->dbeta, "agx_layernorm_bwd2: the second-order pass has no term in beta");
  AGX_CHECK_ARG(p->dx || p->ddy || p->dgamma || p->rows == 0, "agx_layernorm_bwd2: no output wanted");
  if (p->rows > 0) AGX_TRY(check_back(p, true, "agx_layernorm_bwd2"));
  NormArgs a = back_args(p);
  a.u = p->u; a.ldu = p->ldu; a.ddy = p->ddy; a.ldddy = p->ldddy;
  return p->dtype == AGX_F32
             ? launch<BWD2, float>(agx::as_stream(stream), a, p->dgamma, nullptr, p->accumulate_params)
             : launch<BWD2, __bf16>(agx::as_stream(stream), a, p->dgamma, nullptr, p->accumulate_params);
}

extern "C" int64_t agx_op_sizeof(int32_t which) {
  switch (which) {
    case 0: return sizeof(agx_norm_t);
    case 1: return sizeof(agx_orth_t);
    case 2: return sizeof(agx_orth_opts_t);
    case 3: return sizeof(agx_muon_t);
    case 4: return sizeof(agx_muon_opts_t);
    default: return -1;
  }
}
