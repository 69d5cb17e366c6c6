// Orthogonalised updates: Newton-Schulz steps X <- X (a I + b A + c A^2), A = X^T X, on matrices whose smaller side n is
// far below the larger one (a Dense kernel over genes: 18161 x 256).
//
// Algebra.  All iterates are X_0 times polynomials of A_0, which commute, so several steps need the long side only twice:
// with P = aI + bA + cA^2 the next Gram matrix is A P^2 and the product of the steps Q <- Q P; X_k = X_0 Q.  An error of
// A_0 in a direction of tiny singular value grows with every step (by up to a^2 in A), so no more than PHASE steps are
// taken this way: then X Q is formed and its Gram matrix computed anew.  (Five steps on a gradient of a few strong
// directions: 3 + 2 steps are off by 1.5e-6, all five from one Gram matrix by 1e-4, the plain fp32 iteration by 4e-6.)
// Matrices of n x n are symmetric: tiles on and above the diagonal are computed and mirrored.
//
// Products run on the fp16 matrix cores at fp32 accuracy: every operand is split into two fp16 terms, v 2^e = hi + lo (22
// bits), and hi.hi + hi.lo + lo.hi are accumulated in fp32 (lo.lo is below 2^-22 of the product).  e comes from the
// largest |x| for the caller's matrix (first launch) and from a bound on the spectral norm, worked out on the host, for
// everything behind it: entries then stay under 2^14, and those down to 2^-25 of the bound keep all bits.  A bf16 operand
// needs one term only (its 8 bits fit).
//
// Tiles of 64 x 64 by four waves of 32 x 32 (mfma 32x32x16), K in steps of 64 through LDS, next step's global loads in
// flight during the products.
#include "agx_common.h"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr int T = 64, BK = 64, LDK = BK + 8;   // (LDS rows of 144 bytes: 16 rows start in 16 different bank groups)
constexpr int PHASE = 3;                       // steps between two Gram matrices
constexpr int MAXB = 256;                      // partial maxima of one matrix
constexpr int TARGET = 14;                     // scaled entries are below 2^TARGET

// n x n matrix as two fp16 planes of np x np (np: n rounded up to T, zeros behind), value = (hi + lo) 2^-e
struct Planes {
  _Float16 *hi;
  int32_t e, np;
  __device__ __forceinline__ _Float16 *lo() const { return hi + (int64_t)np * np; }
};

__device__ __forceinline__ int exponent_of(uint32_t absbits) {   // e with |v| < 2^e for the float of these bits
  return absbits == 0 ? 0 : (int)(absbits >> 23) - 126;
}
__device__ __forceinline__ void split(float v, _Float16 &hi, _Float16 &lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// ---------------------------------------------------------------------------------------------------------------------
// largest |x|; with a momentum step in front where m is given: m <- mu m + g, u = g + mu m (nesterov) or m
// ---------------------------------------------------------------------------------------------------------------------
struct PrepJob {
  const void *x;        // matrix (g with momentum)
  float *m, *u;         // momentum buffer; where u goes (NULL: u is m)
  int64_t ldx, ldm, ldu;
  int32_t rows, cols, dtype, nb;
  uint32_t *maxb;
};
struct PrepArgs {
  PrepJob job[AGX_MAX_ORTH];
  float mu;
  int nesterov;
};

__global__ __launch_bounds__(256) void orth_prep_kernel(PrepArgs a) {
  const PrepJob j = a.job[blockIdx.y];
  if ((int)blockIdx.x >= j.nb) return;
  __shared__ uint32_t red[4];
  uint32_t mx = 0;
  for (int64_t r = blockIdx.x; r < j.rows; r += j.nb)
    for (int c = threadIdx.x; c < j.cols; c += 256) {
      float v = j.dtype == AGX_F32 ? reinterpret_cast<const float *>(j.x)[r * j.ldx + c]
                                   : (float)reinterpret_cast<const __bf16 *>(j.x)[r * j.ldx + c];
      if (j.m) {
        const float m = a.mu * j.m[r * j.ldm + c] + v;
        j.m[r * j.ldm + c] = m;
        v = a.nesterov ? v + a.mu * m : m;
        if (j.u) j.u[r * j.ldu + c] = v;
      }
      mx = max(mx, __float_as_uint(v) & 0x7fffffffu);   // (as integers: infinities and NaN win)
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
  __syncthreads();
  if (threadIdx.x == 0) j.maxb[blockIdx.x] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// scale exponent of a matrix from its partial maxima; every thread of the 256 gets it
__device__ __forceinline__ int scale_exponent(const uint32_t *maxb, int nb, uint32_t *red) {
  uint32_t mx = (int)threadIdx.x < nb ? maxb[threadIdx.x] : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
  __syncthreads();
  mx = max(max(red[0], red[1]), max(red[2], red[3]));
  return TARGET - exponent_of(mx);
}

// ---------------------------------------------------------------------------------------------------------------------
// tile product: operands in LDS as [64 rows][64 k] fp16 planes
// ---------------------------------------------------------------------------------------------------------------------
struct Tile {
  _Float16 hi[T * LDK], lo[T * LDK];
};

// rows r0.. of a planes matrix, k contiguous (a symmetric matrix: also its columns)
struct LoadPlanes {
  static constexpr bool two = true;
  const _Float16 *hi, *lo;
  int64_t ld;
  half8 v[4];
  __device__ __forceinline__ explicit LoadPlanes(const Planes &m) : hi(m.hi), lo(m.lo()), ld(m.np) {}
  __device__ __forceinline__ void fetch(int r0, int64_t k0) {
    const int row = threadIdx.x >> 3, k = (threadIdx.x & 7) * 8;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t o = (int64_t)(r0 + row + 32 * p) * ld + k0 + k;
      v[2 * p] = *reinterpret_cast<const half8 *>(hi + o);
      v[2 * p + 1] = *reinterpret_cast<const half8 *>(lo + o);
    }
  }
  __device__ __forceinline__ void store(Tile &t) const {
    const int row = threadIdx.x >> 3, k = (threadIdx.x & 7) * 8;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      *reinterpret_cast<half8 *>(&t.hi[(row + 32 * p) * LDK + k]) = v[2 * p];
      *reinterpret_cast<half8 *>(&t.lo[(row + 32 * p) * LDK + k]) = v[2 * p + 1];
    }
  }
};

// rows r0.. of a caller's matrix, k contiguous; zeros outside [rows) x [kmax)
template <typename E> struct LoadK {
  static constexpr bool two = sizeof(E) == 4;
  const E *p;
  int64_t ld, rows, kmax;
  int e;
  float v[4][4];
  __device__ __forceinline__ void fetch(int64_t r0, int64_t k0) {
    const int64_t k = k0 + (threadIdx.x & 15) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t row = r0 + (threadIdx.x >> 4) + 16 * q;
      const E *s = p + row * ld + k;
      if (row < rows && k + 4 <= kmax) {
        if constexpr (sizeof(E) == 4) {
          const f32x4u w = *reinterpret_cast<const f32x4u *>(s);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[q][i] = w[i];
        } else {
          const bf16x4u w = *reinterpret_cast<const bf16x4u *>(s);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[q][i] = (float)w[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[q][i] = row < rows && k + i < kmax ? (float)s[i] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(Tile &t) const {
    const int k = (threadIdx.x & 15) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int row = (threadIdx.x >> 4) + 16 * q;
      half4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        _Float16 h, l;
        split(__builtin_ldexpf(v[q][i], e), h, l);
        hi[i] = h;
        lo[i] = l;
      }
      *reinterpret_cast<half4 *>(&t.hi[row * LDK + k]) = hi;
      if (two) *reinterpret_cast<half4 *>(&t.lo[row * LDK + k]) = lo;
    }
  }
};

// columns r0.. of a caller's matrix whose rows are k: element (r, k) at p[k * ld + r]
template <typename E> struct LoadT {
  static constexpr bool two = sizeof(E) == 4;
  const E *p;
  int64_t ld, rows, kmax;
  int e;
  float v[2][8];
  __device__ __forceinline__ void fetch(int64_t r0, int64_t k0) {
    const int64_t row = r0 + (threadIdx.x & 63);
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t k = k0 + ((threadIdx.x >> 6) + 4 * q) * 8 + i;
        v[q][i] = row < rows && k < kmax ? (float)p[k * ld + row] : 0.f;
      }
  }
  __device__ __forceinline__ void store(Tile &t) const {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int o = (threadIdx.x & 63) * LDK + ((threadIdx.x >> 6) + 4 * q) * 8;
      half8 hi, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        _Float16 h, l;
        split(__builtin_ldexpf(v[q][i], e), h, l);
        hi[i] = h;
        lo[i] = l;
      }
      *reinterpret_cast<half8 *>(&t.hi[o]) = hi;
      if (two) *reinterpret_cast<half8 *>(&t.lo[o]) = lo;
    }
  }
};

// acc = A-tile (rows ra..) . B-tile (rows rb..)^T over k in [k0, k1), k1 - k0 a multiple of BK.  The matrix cores add 64
// k's, vector additions the steps of 64, and the small terms of the split have an accumulator of their own: a long chain
// of additions to one fp32 sum would lose what the split keeps.
template <class LA, class LB>
__device__ __forceinline__ void tile_product(LA &la, LB &lb, int64_t ra, int64_t rb, int64_t k0, int64_t k1, Tile &ta, Tile &tb,
                                             f32x16 &acc) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fa = ((wave >> 1) * 32 + (lane & 31)) * LDK + (lane >> 5) * 8;
  const int fb = ((wave & 1) * 32 + (lane & 31)) * LDK + (lane >> 5) * 8;
  f32x16 cross = {};
  acc = cross;
  la.fetch(ra, k0);
  lb.fetch(rb, k0);
  for (int64_t k = k0; k < k1; k += BK) {
    __syncthreads();
    la.store(ta);
    lb.store(tb);
    __syncthreads();
    if (k + BK < k1) {
      la.fetch(ra, k + BK);
      lb.fetch(rb, k + BK);
    }
    f32x16 sum = {};
#pragma unroll
    for (int s = 0; s < BK; s += 16) {
      const half8 ah = *reinterpret_cast<const half8 *>(&ta.hi[fa + s]);
      const half8 bh = *reinterpret_cast<const half8 *>(&tb.hi[fb + s]);
      sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, sum, 0, 0, 0);
      if constexpr (LB::two) {
        const half8 bl = *reinterpret_cast<const half8 *>(&tb.lo[fb + s]);
        cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, cross, 0, 0, 0);
      }
      if constexpr (LA::two) {
        const half8 al = *reinterpret_cast<const half8 *>(&ta.lo[fa + s]);
        cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, cross, 0, 0, 0);
      }
    }
    acc += sum;
  }
  acc += cross;
}
// accumulator element i of a lane: row frag_row(i) + wave row, column lane & 31 + wave column
__device__ __forceinline__ int frag_row(int i) {
  return ((threadIdx.x >> 7) * 32) + 8 * (i >> 2) + 4 * ((threadIdx.x >> 5) & 1) + (i & 3);
}
__device__ __forceinline__ int frag_col() { return ((threadIdx.x >> 6) & 1) * 32 + (threadIdx.x & 31); }

// ---------------------------------------------------------------------------------------------------------------------
// Gram matrix of the long side, K split over workgroups: partial tiles [tile][slice][64][64] of the scaled matrix
// ---------------------------------------------------------------------------------------------------------------------
struct GramJob {
  const void *x;
  int64_t ld, K, kper;          // K: long side; kper: k of one slice (a multiple of BK)
  int32_t n, nt, slices, tall;  // n: small side, nt: tiles along it; tall: element (i, k) at x[k * ld + i]
  int32_t dtype, e, nb;         // e: scale exponent where nb == 0, otherwise from the partial maxima
  const uint32_t *maxb;
  float *part;
  int32_t first;                // first workgroup of the job
};
struct GramArgs {
  GramJob job[AGX_MAX_ORTH];
  int n;
};

template <class L>
__device__ __forceinline__ void gram_tile(const GramJob &j, int ti, int tj, int64_t k0, int64_t k1, int e, Tile &ta, Tile &tb,
                                          f32x16 &acc) {
  L la, lb;
  la.p = reinterpret_cast<decltype(la.p)>(j.x);
  la.ld = j.ld; la.rows = j.n; la.kmax = j.K; la.e = e;
  lb = la;
  tile_product(la, lb, (int64_t)ti * T, (int64_t)tj * T, k0, k1, ta, tb, acc);
}

__global__ __launch_bounds__(256) void orth_gram_kernel(GramArgs a) {
  __shared__ Tile ta, tb;
  __shared__ uint32_t red[4];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const GramJob &j = a.job[q];
  const int local = blockIdx.x - j.first, tile = local / j.slices, slice = local % j.slices;
  int ti, tj;
  agx::tri_decode(tile, j.nt, ti, tj);
  const int64_t k0 = (int64_t)slice * j.kper, k1 = k0 + j.kper;   // (slices end inside K rounded up; loads stop at K)
  const int e = j.nb ? scale_exponent(j.maxb, j.nb, red) : j.e;
  f32x16 acc;
  if (j.dtype == AGX_F32) {
    if (j.tall) gram_tile<LoadT<float>>(j, ti, tj, k0, k1, e, ta, tb, acc);
    else gram_tile<LoadK<float>>(j, ti, tj, k0, k1, e, ta, tb, acc);
  } else {
    if (j.tall) gram_tile<LoadT<__bf16>>(j, ti, tj, k0, k1, e, ta, tb, acc);
    else gram_tile<LoadK<__bf16>>(j, ti, tj, k0, k1, e, ta, tb, acc);
  }
  float *p = j.part + ((int64_t)tile * j.slices + slice) * T * T;
#pragma unroll
  for (int i = 0; i < 16; ++i) p[frag_row(i) * T + frag_col()] = acc[i];
}

// value (hi + lo) 2^-e of element o of a planes matrix, scaled by 2^e
__device__ __forceinline__ float plane_value(const Planes &m, int64_t o) { return (float)m.hi[o] + (float)m.lo()[o]; }
__device__ __forceinline__ void plane_store(const Planes &m, int64_t o, float scaled) {
  _Float16 h, l;
  split(scaled, h, l);
  m.hi[o] = h;
  m.lo()[o] = l;
}

// An element on or above the diagonal and its mirror image.  Products of matrices that are symmetric up to rounding are not
// symmetric themselves, and the iteration would multiply the difference (rank-deficient matrices: 50 times the error).
__device__ __forceinline__ void store_symmetric(const Planes &m, int64_t r, int64_t c, float scaled) {
  if (r > c) return;
  plane_store(m, r * m.np + c, scaled);
  if (r != c) plane_store(m, c * m.np + r, scaled);
}

// A_0 = (sum of the partial Gram tiles) / d^2 with d = |X|_F + eps (first phase; the scaled matrix's trace is |X|_F^2) or
// without a divisor (later phases).  Every workgroup sums the trace itself, in the same order.
struct ReduceJob {
  const float *part;
  const uint32_t *maxb;
  double *invd;                 // 1 / d of the scaled matrix, for the product with the long side (phase 0)
  Planes A;
  int32_t nt, slices, e, nb, normalise, first;
};
struct ReduceArgs {
  ReduceJob job[AGX_MAX_ORTH];
  int n;
  float eps;
};
__global__ __launch_bounds__(256) void orth_reduce_kernel(ReduceArgs a) {
  __shared__ uint32_t red[4];
  __shared__ double tr[4];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const ReduceJob &j = a.job[q];
  const int tile = blockIdx.x - j.first;
  int ti, tj;
  agx::tri_decode(tile, j.nt, ti, tj);
  double f;
  if (j.normalise) {
    const int e = scale_exponent(j.maxb, j.nb, red);
    double s = 0.0;
    for (int t = 0, id = 0; t < j.nt; id += j.nt - t, ++t)          // diagonal tiles
      for (int z = threadIdx.x; z < j.slices * T; z += 256)
        s += (double)j.part[((int64_t)id * j.slices + z / T) * T * T + (z % T) * (T + 1)];
    s = agx::wave_sum(s);
    if ((threadIdx.x & 63) == 0) tr[threadIdx.x >> 6] = s;
    __syncthreads();
    s = tr[0] + tr[1] + tr[2] + tr[3];
    const double d = sqrt(s) + ldexp((double)a.eps, e);
    const double inv = s == 0.0 ? 0.0 : 1.0 / d;                    // (a matrix of zeros gives zeros)
    f = ldexp(inv * inv, j.A.e);
    if (tile == 0 && threadIdx.x == 0) *j.invd = inv;
  } else {
    f = ldexp(1.0, j.A.e - 2 * j.e);
  }
  for (int z = threadIdx.x; z < T * T; z += 256) {
    float s = 0.f;
    const float *p = j.part + (int64_t)tile * j.slices * T * T + z;
    for (int c = 0; c < j.slices; ++c) s += p[(int64_t)c * T * T];
    const float v = (float)((double)s * f);
    const int64_t r = (int64_t)ti * T + z / T, c = (int64_t)tj * T + z % T;
    store_symmetric(j.A, r, c, v);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// products of the small side: C = alpha L R + beta E + gamma I (L, R, E symmetric and commuting: C symmetric)
// ---------------------------------------------------------------------------------------------------------------------
struct ChainJob {
  Planes L, R, E, C;
  float alpha, beta, gamma;     // beta = 0: E is not read
  int32_t n, nt, first;
};
struct ChainArgs {
  ChainJob job[2 * AGX_MAX_ORTH];
  int n;
};
static_assert(sizeof(ChainArgs) <= 4096, "kernel argument size");

__global__ __launch_bounds__(256) void orth_chain_kernel(ChainArgs a) {
  __shared__ Tile ta, tb;
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const ChainJob &j = a.job[q];
  int ti, tj;
  agx::tri_decode(blockIdx.x - j.first, j.nt, ti, tj);
  LoadPlanes la(j.L), lb(j.R);
  f32x16 acc;
  tile_product(la, lb, ti * T, tj * T, 0, j.C.np, ta, tb, acc);
  // (in 64 bits: near the fixed point a + b + c = 0.7 is what remains of 3.4 - 4.8 + 2.0)
  const double fa = ldexp((double)j.alpha, j.C.e - j.L.e - j.R.e);
  const double fb = ldexp((double)j.beta, j.C.e - j.E.e), fi = ldexp((double)j.gamma, j.C.e);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t r = (int64_t)ti * T + frag_row(i), c = (int64_t)tj * T + frag_col(), o = r * j.C.np + c;
    double w = fa * (double)acc[i];
    if (j.beta != 0.f) w += fb * (double)plane_value(j.E, o);
    if (r == c && r < j.n) w += fi;
    const float v = (float)w;
    store_symmetric(j.C, r, c, v);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// product with the long side: Y = X Q / d, or from the left for a wide matrix
// ---------------------------------------------------------------------------------------------------------------------
struct ApplyJob {
  const void *x;
  void *out;                    // result of dtype `otype`, or the weights of a Muon step
  int64_t ldx, ldo;
  Planes Q;
  const uint32_t *maxb;
  const double *invd;           // NULL: no divisor
  float decay, step;            // a Muon step: out <- decay * out - step * Y
  int32_t rows, cols, tall, dtype, otype, e, nb, tc, muon, first;   // tc: tiles along the columns
};
struct ApplyArgs {
  ApplyJob job[AGX_MAX_ORTH];
  int n;
};

template <typename E>
__device__ __forceinline__ void apply_tile(const ApplyJob &j, int tr, int tc, int e, Tile &ta, Tile &tb, f32x16 &acc) {
  LoadPlanes lq(j.Q);
  if (j.tall) {
    LoadK<E> lx;
    lx.p = reinterpret_cast<const E *>(j.x); lx.ld = j.ldx; lx.rows = j.rows; lx.kmax = j.cols; lx.e = e;
    tile_product(lx, lq, (int64_t)tr * T, (int64_t)tc * T, 0, j.Q.np, ta, tb, acc);
  } else {
    LoadT<E> lx;
    lx.p = reinterpret_cast<const E *>(j.x); lx.ld = j.ldx; lx.rows = j.cols; lx.kmax = j.rows; lx.e = e;
    tile_product(lq, lx, (int64_t)tr * T, (int64_t)tc * T, 0, j.Q.np, ta, tb, acc);
  }
}

__global__ __launch_bounds__(256) void orth_apply_kernel(ApplyArgs a) {
  __shared__ Tile ta, tb;
  __shared__ uint32_t red[4];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const ApplyJob &j = a.job[q];
  const int tr = (blockIdx.x - j.first) / j.tc, tc = (blockIdx.x - j.first) % j.tc;
  const int e = j.nb ? scale_exponent(j.maxb, j.nb, red) : j.e;
  f32x16 acc;
  if (j.dtype == AGX_F32) apply_tile<float>(j, tr, tc, e, ta, tb, acc);
  else apply_tile<__bf16>(j, tr, tc, e, ta, tb, acc);
  // (in 64 bits: 1 / d spans more than fp32's exponents for tiny matrices)
  const double f = ldexp(j.invd ? *j.invd : ldexp(1.0, -e), -j.Q.e);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t r = (int64_t)tr * T + frag_row(i), c = (int64_t)tc * T + frag_col();
    if (r >= j.rows || c >= j.cols) continue;
    const float y = (float)((double)acc[i] * f);
    if (j.muon) {
      float *w = reinterpret_cast<float *>(j.out) + r * j.ldo + c;
      *w = j.decay * *w - j.step * y;
    } else if (j.otype == AGX_F32) {
      reinterpret_cast<float *>(j.out)[r * j.ldo + c] = y;
    } else {
      reinterpret_cast<__bf16 *>(j.out)[r * j.ldo + c] = (__bf16)y;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
struct Job {          // one matrix of a call
  const void *x;      // what is orthogonalised (g of a Muon job without nesterov and momentum: see run())
  void *out;
  int64_t ldx, ldo;
  int rows, cols, dtype;
  // Muon
  float *m = nullptr;
  int64_t ldm = 0;
  float decay = 0.f, step = 0.f;
  bool muon = false;
  bool tall() const { return rows >= cols; }
  int n() const { return std::min(rows, cols); }
  int64_t K() const { return std::max(rows, cols); }
  int nt() const { return agx::cdiv(n(), T); }
  int np() const { return nt() * T; }
};

struct Layout {       // workspace of one job, in bytes from its start
  int64_t maxb, invd, mat[5], part, x[2], u, end;
  int slices;
  int64_t kper;
};
int64_t up256(int64_t v) { return (v + 255) & ~(int64_t)255; }

// slices of a Gram product: about three workgroups a CU over all of the call's matrices
void plan(const Job &j, int total_tiles, int phases, bool need_u, Layout &l) {
  const int tiles = j.nt() * (j.nt() + 1) / 2;
  const int64_t ksteps = agx::cdiv64(j.K(), BK);
  const int64_t want = std::max<int64_t>(1, (int64_t)agx::num_cus() * 3 / std::max(1, total_tiles));
  l.kper = agx::cdiv64(ksteps, std::min(ksteps, want)) * BK;
  l.slices = (int)agx::cdiv64(j.K(), l.kper);
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = up256(off + bytes); return o; };
  l.maxb = take(MAXB * 4);
  l.invd = take(8);
  for (int64_t &m : l.mat) m = take((int64_t)j.np() * j.np() * 4);
  l.part = take((int64_t)tiles * l.slices * T * T * 4);
  for (int k = 0; k < 2; ++k) l.x[k] = phases > 1 + k ? take((int64_t)j.rows * j.cols * 4) : 0;
  l.u = need_u ? take((int64_t)j.rows * j.cols * 4) : 0;
  l.end = off;
}
int phases_of(int steps) { return agx::cdiv(steps, PHASE); }

int64_t ws_bytes(const Job *jobs, int n, int steps, bool need_u) {
  int tiles = 0;
  for (int i = 0; i < n; ++i) tiles += jobs[i].nt() * (jobs[i].nt() + 1) / 2;
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    Layout l;
    plan(jobs[i], tiles, phases_of(steps), need_u, l);
    total += l.end;
  }
  return total;
}

// Bounds on the spectral norms of a step's matrices where the iterate's singular values are at most s: |a s + b s^3 + c s^5|
// and its parts over [0, s], by the polynomials' stationary points (of the even polynomials in lambda = s^2).
struct Bounds {
  double P, S, next;   // P = a + bA + cA^2, S = A P, next: s of the next iterate
};
Bounds bounds_of(double s, double a, double b, double c) {
  const double L = s * s;
  auto worst = [&](auto f, const double *at, int n) {
    double w = std::max(std::fabs(f(0.0)), std::fabs(f(L)));
    for (int i = 0; i < n; ++i)
      if (at[i] > 0.0 && at[i] < L) w = std::max(w, std::fabs(f(at[i])));
    return w;
  };
  Bounds r;
  const double p1[1] = {c != 0.0 ? -b / (2.0 * c) : -1.0};
  r.P = worst([&](double x) { return a + b * x + c * x * x; }, p1, 1);
  auto roots = [](double p, double q, double w, double *out) {   // p + q x + w x^2 = 0
    if (w == 0.0) { out[0] = q != 0.0 ? -p / q : -1.0; out[1] = -1.0; return; }
    const double d = q * q - 4.0 * w * p;
    if (d < 0.0) { out[0] = out[1] = -1.0; return; }
    out[0] = (-q + std::sqrt(d)) / (2.0 * w);
    out[1] = (-q - std::sqrt(d)) / (2.0 * w);
  };
  double z[2];
  roots(a, 2.0 * b, 3.0 * c, z);
  r.S = worst([&](double x) { return x * (a + b * x + c * x * x); }, z, 2);
  roots(a, 3.0 * b, 5.0 * c, z);
  r.next = worst([&](double x) { return std::sqrt(x) * (a + b * x + c * x * x); }, z, 2);
  return r;
}
// scale exponent of a matrix whose entries are bounded: half of the range is kept for rounding beyond the bound
int exponent_for(double bound) {
  if (!(bound > 0.0)) return 0;
  return TARGET - (std::ilogb(bound) + 1);
}

int check_opts(const agx_orth_opts_t *o, const char *who) {
  AGX_CHECK_ARG(o, "%s: options missing", who);
  AGX_CHECK_ARG(o->steps >= 1 && o->steps <= AGX_ORTH_MAX_STEPS, "%s: steps %d outside 1..%d", who, o->steps, AGX_ORTH_MAX_STEPS);
  AGX_CHECK_ARG(o->n_coef == 1 || o->n_coef == o->steps, "%s: %d coefficient triples for %d steps", who, o->n_coef, o->steps);
  AGX_CHECK_ARG(o->eps >= 0.f && std::isfinite(o->eps), "%s: eps must be finite and not negative", who);
  double s = 1.0;
  for (int k = 0; k < o->steps; ++k) {
    const float *c = o->coef + (o->n_coef == 1 ? 0 : 3 * k);
    AGX_CHECK_ARG(std::isfinite(c[0]) && std::isfinite(c[1]) && std::isfinite(c[2]), "%s: coefficients must be finite", who);
    s = bounds_of(s, c[0], c[1], c[2]).next;
    AGX_CHECK_ARG(s > 1e-3 && s < 1e3, "%s: with these coefficients singular values in [0, 1] reach %g after step %d", who, s, k + 1);
  }
  return AGX_OK;
}

int run(hipStream_t st, Job *jobs, int n, const agx_orth_opts_t *o, float mu, bool nesterov, char *ws, int64_t bytes,
        const char *who) {
  const bool need_u = mu != 0.f && nesterov;   // (jobs of one call are all Muon jobs or none is)
  const int64_t need = ws_bytes(jobs, n, o->steps, need_u && jobs[0].muon);
  if (!ws || bytes < need) {
    agx::set_error("%s: workspace of %lld bytes, %lld needed", who, (long long)bytes, (long long)need);
    return AGX_E_WORKSPACE;
  }
  AGX_CHECK_ARG(agx::aligned16(ws), "%s: workspace must be 16-byte aligned", who);
  int tiles = 0;
  for (int i = 0; i < n; ++i) tiles += jobs[i].nt() * (jobs[i].nt() + 1) / 2;
  const int phases = phases_of(o->steps);
  Layout lay[AGX_MAX_ORTH];
  char *base[AGX_MAX_ORTH];
  int nb[AGX_MAX_ORTH];
  {
    PrepArgs pa;
    memset(&pa, 0, sizeof(pa));
    pa.mu = mu;
    pa.nesterov = nesterov;
    int gx = 1;
    for (int i = 0; i < n; ++i) {
      Job &j = jobs[i];
      plan(j, tiles, phases, need_u && j.muon, lay[i]);
      base[i] = ws;
      ws += lay[i].end;
      nb[i] = std::min(MAXB, j.rows);
      gx = std::max(gx, nb[i]);
      PrepJob &p = pa.job[i];
      p.x = j.x; p.ldx = j.ldx; p.rows = j.rows; p.cols = j.cols; p.dtype = j.dtype; p.nb = nb[i];
      p.maxb = reinterpret_cast<uint32_t *>(base[i] + lay[i].maxb);
      if (j.muon) {
        p.m = j.m;
        p.ldm = j.ldm;
        if (need_u) {
          p.u = reinterpret_cast<float *>(base[i] + lay[i].u);
          p.ldu = j.cols;
          j.x = p.u;
          j.ldx = j.cols;
        } else {
          j.x = j.m;
          j.ldx = j.ldm;
        }
      }
    }
    hipLaunchKernelGGL(orth_prep_kernel, dim3(gx, n), dim3(256), 0, st, pa);
    AGX_LAUNCH_CHECK();
  }
  const void *x[AGX_MAX_ORTH];
  int64_t ldx[AGX_MAX_ORTH];
  for (int i = 0; i < n; ++i) { x[i] = jobs[i].x; ldx[i] = jobs[i].ldx; }
  auto planes = [&](int i, int k, int e) {
    Planes p;
    p.hi = reinterpret_cast<_Float16 *>(base[i] + lay[i].mat[k]);
    p.e = e;
    p.np = jobs[i].np();
    return p;
  };
  double s = 1.0;       // bound on the iterate's singular values (|X_0| <= |X_0|_F <= 1)
  for (int ph = 0, k = 0; ph < phases; ++ph) {
    const bool first = ph == 0, last = ph == phases - 1;
    const int ex = exponent_for(s);                 // scale of the iterate (later phases)
    {
      GramArgs ga;
      ReduceArgs ra;
      ga.n = ra.n = n;
      ra.eps = o->eps;
      int gb = 0, rb = 0;
      for (int i = 0; i < n; ++i) {
        const Job &j = jobs[i];
        const Layout &l = lay[i];
        const int nt = j.nt(), tl = nt * (nt + 1) / 2;
        GramJob &g = ga.job[i];
        g.x = x[i]; g.ld = ldx[i]; g.K = j.K(); g.kper = l.kper; g.n = j.n(); g.nt = nt; g.slices = l.slices; g.tall = j.tall();
        g.dtype = first ? j.dtype : AGX_F32; g.e = ex; g.nb = first ? nb[i] : 0;
        g.maxb = reinterpret_cast<const uint32_t *>(base[i] + l.maxb);
        g.part = reinterpret_cast<float *>(base[i] + l.part);
        g.first = gb;
        gb += tl * l.slices;
        ReduceJob &r = ra.job[i];
        r.part = g.part; r.maxb = g.maxb; r.invd = reinterpret_cast<double *>(base[i] + l.invd);
        r.A = planes(i, 0, exponent_for(s * s)); r.nt = nt; r.slices = l.slices; r.e = ex; r.nb = nb[i];
        r.normalise = first; r.first = rb;
        rb += tl;
      }
      hipLaunchKernelGGL(orth_gram_kernel, dim3(gb), dim3(256), 0, st, ga);
      AGX_LAUNCH_CHECK();
      hipLaunchKernelGGL(orth_reduce_kernel, dim3(rb), dim3(256), 0, st, ra);
      AGX_LAUNCH_CHECK();
    }
    // matrices: 0 A, 1 P, 2 A P, 3 / 4 Q
    const int steps = std::min(PHASE, o->steps - k);
    double bQ = 1.0;                                // |Q| <= bQ
    int iq = 3, eA = exponent_for(s * s), eQ = 0;
    for (int t = 0; t < steps; ++t, ++k) {
      const float *c = o->coef + (o->n_coef == 1 ? 0 : 3 * k);
      const Bounds b = bounds_of(s, c[0], c[1], c[2]);
      const int eP = exponent_for(b.P), eS = exponent_for(b.S), eN = exponent_for(b.next * b.next);
      const int iP = t == 0 ? iq : 1;               // the first step's P is Q too
      bQ *= b.P;
      const int eQn = exponent_for(bQ);
      auto launch = [&](int per, auto fill) -> int {
        ChainArgs ca;
        int blocks = 0;
        ca.n = n * per;
        for (int i = 0; i < n; ++i)
          for (int w = 0; w < per; ++w) {
            ChainJob &g = ca.job[i * per + w];
            memset(&g, 0, sizeof(g));
            g.n = jobs[i].n(); g.nt = jobs[i].nt(); g.first = blocks; g.alpha = 1.f;
            blocks += g.nt * (g.nt + 1) / 2;
            fill(g, i, w);
          }
        hipLaunchKernelGGL(orth_chain_kernel, dim3(blocks), dim3(256), 0, st, ca);
        AGX_LAUNCH_CHECK();
        return AGX_OK;
      };
      AGX_TRY(launch(1, [&](ChainJob &g, int i, int) {               // P = a I + b A + c A^2
        g.L = g.R = g.E = planes(i, 0, eA);
        g.C = planes(i, iP, eP);
        g.alpha = c[2]; g.beta = c[1]; g.gamma = c[0];
      }));
      const bool more = t + 1 < steps;
      const int two = (more ? 1 : 0) + (t > 0 ? 1 : 0);
      if (two)
        AGX_TRY(launch(two, [&](ChainJob &g, int i, int w) {         // S = A P (where a step follows) | Q <- Q P
          const bool sp = more && w == 0;
          g.R = planes(i, iP, eP);
          g.L = sp ? planes(i, 0, eA) : planes(i, iq, eQ);
          g.C = sp ? planes(i, 2, eS) : planes(i, 7 - iq, eQn);
        }));
      if (t > 0) iq = 7 - iq;
      eQ = eQn;
      if (more)
        AGX_TRY(launch(1, [&](ChainJob &g, int i, int) {             // A <- S P
          g.L = planes(i, 2, eS);
          g.R = planes(i, iP, eP);
          g.C = planes(i, 0, eN);
        }));
      eA = eN;
      s = b.next;
    }
    ApplyArgs aa;
    aa.n = n;
    int blocks = 0;
    for (int i = 0; i < n; ++i) {
      const Job &j = jobs[i];
      ApplyJob &g = aa.job[i];
      memset(&g, 0, sizeof(g));
      g.x = x[i]; g.ldx = ldx[i]; g.Q = planes(i, iq, eQ);
      g.maxb = reinterpret_cast<const uint32_t *>(base[i] + lay[i].maxb);
      g.invd = first ? reinterpret_cast<const double *>(base[i] + lay[i].invd) : nullptr;
      g.rows = j.rows; g.cols = j.cols; g.tall = j.tall();
      g.dtype = first ? j.dtype : AGX_F32; g.e = ex; g.nb = first ? nb[i] : 0;
      if (last) {
        g.out = j.out; g.ldo = j.ldo; g.otype = j.dtype; g.muon = j.muon; g.decay = j.decay; g.step = j.step;
      } else {
        g.out = base[i] + lay[i].x[ph & 1]; g.ldo = j.cols; g.otype = AGX_F32;
        x[i] = g.out;
        ldx[i] = g.ldo;
      }
      g.tc = agx::cdiv(j.cols, T);
      g.first = blocks;
      blocks += agx::cdiv(j.rows, T) * g.tc;
    }
    hipLaunchKernelGGL(orth_apply_kernel, dim3(blocks), dim3(256), 0, st, aa);
    AGX_LAUNCH_CHECK();
  }
  return AGX_OK;
}

int to_jobs(const agx_orth_t *j, int n, Job *out, const char *who) {
  AGX_CHECK_ARG(j && n >= 1 && n <= AGX_MAX_ORTH, "%s: 1 to %d matrices a call", who, AGX_MAX_ORTH);
  for (int i = 0; i < n; ++i) {
    const agx_orth_t &a = j[i];
    AGX_CHECK_ARG(a.dtype == AGX_F32 || a.dtype == AGX_BF16, "%s: matrix %d: dtype %d", who, i, a.dtype);
    AGX_CHECK_ARG(a.rows > 0 && a.cols > 0 && std::min(a.rows, a.cols) <= AGX_ORTH_MAX_SIDE,
                  "%s: matrix %d is %d x %d; the smaller side is at most %d", who, i, a.rows, a.cols, AGX_ORTH_MAX_SIDE);
    AGX_CHECK_ARG(agx::cdiv64(a.rows, T) * agx::cdiv64(a.cols, T) < (1 << 26), "%s: matrix %d is too large", who, i);
    Job &b = out[i];
    b.x = a.x; b.out = a.out; b.ldx = a.ldx; b.ldo = a.ldo; b.rows = a.rows; b.cols = a.cols; b.dtype = a.dtype;
  }
  return AGX_OK;
}

int muon_jobs(const agx_muon_t *j, int n, const agx_muon_opts_t *o, Job *out, const char *who) {
  AGX_CHECK_ARG(j && n >= 1 && n <= AGX_MAX_ORTH, "%s: 1 to %d matrices a call", who, AGX_MAX_ORTH);
  agx_orth_t m[AGX_MAX_ORTH];
  memset(m, 0, sizeof(m));
  for (int i = 0; i < n; ++i) {
    m[i].x = j[i].g; m[i].ldx = j[i].ldg; m[i].out = j[i].w; m[i].ldo = j[i].ldw;
    m[i].rows = j[i].rows; m[i].cols = j[i].cols; m[i].dtype = AGX_F32;
  }
  AGX_TRY(to_jobs(m, n, out, who));
  for (int i = 0; i < n; ++i) {
    out[i].muon = true;
    out[i].m = j[i].m;
    out[i].ldm = j[i].ldm;
    out[i].decay = 1.f - o->lr * o->weight_decay;
    out[i].step = o->lr * j[i].scale;
  }
  return AGX_OK;
}

}  // namespace

extern "C" int64_t agx_orth_ws_bytes(const agx_orth_t *jobs, int32_t n, int32_t steps) {
  Job j[AGX_MAX_ORTH];
  if (steps < 1 || steps > AGX_ORTH_MAX_STEPS || to_jobs(jobs, n, j, "agx_orth_ws_bytes") != AGX_OK) return -1;
  return ws_bytes(j, n, steps, false);
}

extern "C" int agx_orthogonalize(void *stream, const agx_orth_t *jobs, int32_t n, const agx_orth_opts_t *o, void *ws,
                                 int64_t ws_size) {
  const char *who = "agx_orthogonalize";
  Job j[AGX_MAX_ORTH];
  AGX_TRY(check_opts(o, who));
  AGX_TRY(to_jobs(jobs, n, j, who));
  for (int i = 0; i < n; ++i) {
    const uintptr_t al = j[i].dtype == AGX_F32 ? 3 : 1;
    AGX_CHECK_ARG(j[i].x && j[i].out && j[i].ldx >= j[i].cols && j[i].ldo >= j[i].cols, "%s: matrix %d: null or leading dimension", who, i);
    AGX_CHECK_ARG(((reinterpret_cast<uintptr_t>(j[i].x) | reinterpret_cast<uintptr_t>(j[i].out)) & al) == 0,
                  "%s: matrix %d not aligned to its elements", who, i);
    AGX_CHECK_ARG(j[i].x != j[i].out, "%s: matrix %d: the result cannot be written over the input", who, i);
  }
  return run(agx::as_stream(stream), j, n, o, 0.f, false, static_cast<char *>(ws), ws_size, who);
}

extern "C" int64_t agx_opt_muon_ws_bytes(const agx_muon_t *jobs, int32_t n, const agx_muon_opts_t *o) {
  const char *who = "agx_opt_muon_ws_bytes";
  if (!o || o->orth.steps < 1 || o->orth.steps > AGX_ORTH_MAX_STEPS) {
    agx::set_error("%s: options missing or steps out of range", who);
    return -1;
  }
  Job j[AGX_MAX_ORTH];
  if (muon_jobs(jobs, n, o, j, who) != AGX_OK) return -1;
  return ws_bytes(j, n, o->orth.steps, o->nesterov && o->momentum != 0.f);
}

extern "C" int agx_opt_muon(void *stream, const agx_muon_t *jobs, int32_t n, const agx_muon_opts_t *o, void *ws, int64_t ws_size) {
  const char *who = "agx_opt_muon";
  AGX_CHECK_ARG(o, "%s: options missing", who);
  AGX_TRY(check_opts(&o->orth, who));
  AGX_CHECK_ARG(o->momentum >= 0.f && o->momentum < 1.f, "%s: momentum must be in [0, 1)", who);
  AGX_CHECK_ARG(std::isfinite(o->lr) && std::isfinite(o->weight_decay), "%s: learning rate / weight decay must be finite", who);
  Job j[AGX_MAX_ORTH];
  AGX_TRY(muon_jobs(jobs, n, o, j, who));
  for (int i = 0; i < n; ++i) {
    const agx_muon_t &a = jobs[i];
    AGX_CHECK_ARG(a.w && a.g && a.m && a.ldw >= a.cols && a.ldg >= a.cols && a.ldm >= a.cols && std::isfinite(a.scale),
                  "%s: matrix %d: null, leading dimension or scale", who, i);
    AGX_CHECK_ARG(((reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.g) | reinterpret_cast<uintptr_t>(a.m)) & 3) == 0,
                  "%s: matrix %d not aligned to its elements", who, i);
    AGX_CHECK_ARG(a.w != a.m && a.w != a.g && a.g != a.m, "%s: matrix %d: w, g and m must be different arrays", who, i);
  }
  return run(agx::as_stream(stream), j, n, &o->orth, o->momentum, o->nesterov != 0, static_cast<char *>(ws), ws_size, who);
}
