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
#include <type_traits>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr int T = 64, BK = 64, LDK = BK + 8;   // (LDS rows of 144 bytes: 16 rows start in 16 different bank groups)
constexpr int PHASE = 3;                       // steps between two Gram matrices
constexpr int MAXB = 1024;                     // partial maxima of one matrix
constexpr int ONE_BLOCK = 128;                 // largest padded side for a phase in one workgroup (LDS)
constexpr int SMALL = 512;                     // largest padded side for the chain's latency form
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
// v = hi + lo, each rounded to nearest
__device__ __forceinline__ void split(float v, _Float16 &hi, _Float16 &lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}
__device__ __forceinline__ void split4(f32x4 v, half4 &hi, half4 &lo) {   // (two values an instruction)
  hi = __builtin_convertvector(v, half4);
  lo = __builtin_convertvector(v - __builtin_convertvector(hi, f32x4), half4);
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

// four consecutive values of a row (n of them valid)
__device__ __forceinline__ void load4(const float *p, int n, float (&v)[4]) {
  if (n == 4) {
    const f32x4u w = *reinterpret_cast<const f32x4u *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}
__device__ __forceinline__ void load4(const __bf16 *p, int n, float (&v)[4]) {
  if (n == 4) {
    const bf16x4u w = *reinterpret_cast<const bf16x4u *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  }
}
__device__ __forceinline__ void store4(float *p, int n, const float (&v)[4]) {
  if (n == 4) {
    f32x4u w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i];
    *reinterpret_cast<f32x4u *>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
}

__global__ __launch_bounds__(256) void orth_prep_kernel(PrepArgs a) {
  const PrepJob j = a.job[blockIdx.y];
  if ((int)blockIdx.x >= j.nb) return;
  __shared__ uint32_t red[4];
  uint32_t mx = 0;
  const uint32_t per_row = (uint32_t)(j.cols + 3) / 4;               // (host: rows * per_row < 2^31)
  const uint32_t items = per_row * (uint32_t)j.rows, step = (uint32_t)j.nb * 256;
#pragma unroll 4
  for (uint32_t it = blockIdx.x * 256 + threadIdx.x; it < items; it += step) {
    const uint32_t r = it / per_row;
    const int c = (int)(it - r * per_row) * 4, n = min(4, j.cols - c);
    float v[4];
    if (j.dtype == AGX_F32) load4(reinterpret_cast<const float *>(j.x) + (int64_t)r * j.ldx + c, n, v);
    else load4(reinterpret_cast<const __bf16 *>(j.x) + (int64_t)r * j.ldx + c, n, v);
    if (j.m) {
      float m[4];
      load4(j.m + (int64_t)r * j.ldm + c, n, m);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = a.mu * m[i] + v[i];
        v[i] = a.nesterov ? v[i] + a.mu * m[i] : m[i];
      }
      store4(j.m + (int64_t)r * j.ldm + c, n, m);
      if (j.u) store4(j.u + (int64_t)r * j.ldu + c, n, v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);   // (as integers: infinities and NaN win)
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
  __syncthreads();
  if (threadIdx.x == 0) j.maxb[blockIdx.x] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// tile (ti <= tj) of linear index t over the upper triangle of nt x nt tiles (nt is small: no square root)
__device__ __forceinline__ void upper_tile(int t, int nt, int &ti, int &tj) {
  ti = 0;
  while (t >= nt - ti) t -= nt - ti++;
  tj = ti + t;
}

// scale exponent of a matrix from its partial maxima; every thread of the 256 gets it
__device__ __forceinline__ int scale_exponent(const uint32_t *maxb, int nb, uint32_t *red) {
  uint32_t mx = 0;
  for (int i = threadIdx.x; i < nb; i += 256) mx = max(mx, maxb[i]);
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
      f32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __builtin_ldexpf(v[q][i], e);
      split4(w, hi, lo);
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
      half4 hi[2], lo[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_ldexpf(v[q][4 * p + i], e);
        split4(w, hi[p], lo[p]);
      }
      *reinterpret_cast<half8 *>(&t.hi[o]) = __builtin_shufflevector(hi[0], hi[1], 0, 1, 2, 3, 4, 5, 6, 7);
      if (two) *reinterpret_cast<half8 *>(&t.lo[o]) = __builtin_shufflevector(lo[0], lo[1], 0, 1, 2, 3, 4, 5, 6, 7);
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
  float *part, *trace;          // trace[ti * slices + slice]: sums of the diagonal of the partial diagonal tiles
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
  __shared__ float tr[4];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const GramJob &j = a.job[q];
  const int local = blockIdx.x - j.first, tile = local / j.slices, slice = local % j.slices;
  int ti, tj;
  upper_tile(tile, j.nt, ti, tj);
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
  if (ti == tj) {
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) d += frag_row(i) == frag_col() ? acc[i] : 0.f;
    d = agx::wave_sum(d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tr[threadIdx.x >> 6] = d;
    __syncthreads();
    if (threadIdx.x == 0) j.trace[ti * j.slices + slice] = tr[0] + tr[1] + tr[2] + tr[3];
  }
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

// A lane's four rows r.. of column c of a 32 x 32 tile, and their mirror image, into planes of row stride ld (global memory
// or LDS).  The mirror image is contiguous; the rows themselves go out as pairs of columns, which two neighbouring lanes
// exchange (the even one takes the first two rows, the odd one the others).  A tile on the diagonal comes symmetric: its
// mirror image is all of it.
__device__ __forceinline__ void store_planes4(_Float16 *hi, _Float16 *lo, int ld, int r, int c, bool diag, f32x4 v) {
  half4 h, l;
  split4(v, h, l);
  *reinterpret_cast<half4 *>(&hi[c * ld + r]) = h;
  *reinterpret_cast<half4 *>(&lo[c * ld + r]) = l;
  if (diag) return;                                    // (uniform over the wave)
  const bool odd = threadIdx.x & 1;
  auto pairs = [&](half4 x, _Float16 *p) {
    const uint2 w = __builtin_bit_cast(uint2, x);      // rows (0, 1) and (2, 3) of this lane's column
    const uint32_t mine = odd ? w.y : w.x, give = odd ? w.x : w.y;
    const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0xb1, 0xf, 0xf, true);   // lanes 2 k <-> 2 k + 1
    const uint32_t a = odd ? got : mine, b = odd ? mine : got;
    uint32_t *q = reinterpret_cast<uint32_t *>(p + (r + (odd ? 2 : 0)) * ld + (c & ~1));
    q[0] = (a & 0xffffu) | (b << 16);
    *reinterpret_cast<uint32_t *>(reinterpret_cast<_Float16 *>(q) + ld) = (a >> 16) | (b & 0xffff0000u);
  };
  pairs(h, hi);
  pairs(l, lo);
}

constexpr int RCH = T * T / 256;   // workgroups a tile
// A_0 = (sum of the partial Gram tiles) / d^2 with d = |X|_F + eps (first phase; the scaled matrix's trace is |X|_F^2) or
// without a divisor (later phases).  Every workgroup sums the trace itself, in the same order.
struct ReduceJob {
  const float *part, *trace;
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
  const int tile = (blockIdx.x - j.first) / RCH, z = (blockIdx.x - j.first) % RCH * 256 + threadIdx.x;
  int ti, tj;
  upper_tile(tile, j.nt, ti, tj);
  float sum = 0.f;
  const float *p = j.part + (int64_t)tile * j.slices * T * T + z;
#pragma unroll 8
  for (int c = 0; c < j.slices; ++c) sum += p[(int64_t)c * T * T];
  double f;
  if (j.normalise) {
    const int e = scale_exponent(j.maxb, j.nb, red);
    double s = 0.0;
    for (int i = threadIdx.x; i < j.nt * j.slices; i += 256) s += (double)j.trace[i];
    s = agx::wave_sum(s);
    if ((threadIdx.x & 63) == 0) tr[threadIdx.x >> 6] = s;
    __syncthreads();
    s = tr[0] + tr[1] + tr[2] + tr[3];
    const double d = sqrt(s) + ldexp((double)a.eps, e);
    const double inv = s == 0.0 ? 0.0 : 1.0 / d;                    // (a matrix of zeros gives zeros)
    f = ldexp(inv * inv, j.A.e);
    if (blockIdx.x == j.first && threadIdx.x == 0) *j.invd = inv;
  } else {
    f = ldexp(1.0, j.A.e - 2 * j.e);
  }
  store_symmetric(j.A, (int64_t)ti * T + z / T, (int64_t)tj * T + z % T, (float)((double)sum * f));
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
  upper_tile(blockIdx.x - j.first, j.nt, ti, tj);
  LoadPlanes la(j.L), lb(j.R);
  f32x16 acc;
  tile_product(la, lb, ti * T, tj * T, 0, j.C.np, ta, tb, acc);
  const float fa = __builtin_ldexpf(j.alpha, j.C.e - j.L.e - j.R.e);
  const float fb = __builtin_ldexpf(j.beta, j.C.e - j.E.e), fi = __builtin_ldexpf(j.gamma, j.C.e);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t r = (int64_t)ti * T + frag_row(i), c = (int64_t)tj * T + frag_col(), o = r * j.C.np + c;
    float w = r == c && r < j.n ? fi : 0.f;
    if (j.beta != 0.f) w = fmaf(fb, plane_value(j.E, o), w);
    const float v = fmaf(fa, acc[i], w);
    store_symmetric(j.C, r, c, v);
  }
}

// The same for small matrices, where a launch is all latency: tiles of 32 x 32 (36 of them at n = 256), k dealt to the four
// waves in blocks of 32, operands straight from L2 to the matrix cores' registers - every load of a wave's k range is
// in flight at once up to n = 256 - and the waves' sums met in LDS.
// (k runs in an order of its own, the same for both operands: a lane's two vectors of a block are neighbours in memory)
__global__ __launch_bounds__(256) void orth_chain_small_kernel(ChainArgs a) {
  __shared__ float part[4][16][64];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const ChainJob &j = a.job[q];
  const int np = j.C.np, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int ti, tj;
  upper_tile(blockIdx.x - j.first, np / 32, ti, tj);
  const int64_t oa = (int64_t)(ti * 32 + (lane & 31)) * np + (lane >> 5) * 16, ob = (int64_t)(tj * 32 + (lane & 31)) * np + (lane >> 5) * 16;
  const _Float16 *ah = j.L.hi + oa, *al = j.L.lo() + oa, *bh = j.R.hi + ob, *bl = j.R.lo() + ob;
  auto at = [](const _Float16 *p, int k) { return *reinterpret_cast<const half8 *>(p + k); };
  const int r = ti * 32 + 8 * wave + 4 * (lane >> 5), c = tj * 32 + (lane & 31);   // the four elements this lane finishes
  float ev[4] = {};
  if (j.beta != 0.f)
  {                                                    // (E is symmetric: its mirror image is one vector)
    const half4 eh = *reinterpret_cast<const half4 *>(&j.E.hi[c * np + r]), el = *reinterpret_cast<const half4 *>(&j.E.lo()[c * np + r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) ev[i] = (float)eh[i] + (float)el[i];
  }
  f32x16 sum = {}, cross = {};
  for (int k = wave * 32; k < np; k += 256) {          // two blocks of 32 a turn
    half8 v[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (k + 128 * h < np) {
        const int o = k + 128 * h;
        v[h][0] = at(ah, o); v[h][1] = at(ah, o + 8); v[h][2] = at(al, o); v[h][3] = at(al, o + 8);
        v[h][4] = at(bh, o); v[h][5] = at(bh, o + 8); v[h][6] = at(bl, o); v[h][7] = at(bl, o + 8);
      }
    f32x16 s = {};
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (k + 128 * h < np) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[h][i], v[h][4 + i], s, 0, 0, 0);
          cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[h][i], v[h][6 + i], cross, 0, 0, 0);
          cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[h][2 + i], v[h][4 + i], cross, 0, 0, 0);
        }
      }
    sum += s;
  }
  sum += cross;
#pragma unroll
  for (int i = 0; i < 16; ++i) part[wave][i][lane] = sum[i];
  __syncthreads();
  const float fa = __builtin_ldexpf(j.alpha, j.C.e - j.L.e - j.R.e);
  const float fb = __builtin_ldexpf(j.beta, j.C.e - j.E.e), fi = __builtin_ldexpf(j.gamma, j.C.e);
  f32x4 out;
  auto total = [&](int f, int l) { return part[0][f][l] + part[1][f][l] + part[2][f][l] + part[3][f][l]; };
#pragma unroll
  for (int i = 0; i < 4; ++i)                          // accumulator element f: row 8 (f / 4) + 4 (lane / 32) + f % 4
    out[i] = fmaf(fa, total(wave * 4 + i, lane), fmaf(fb, ev[i], r + i == c && c < j.n ? fi : 0.f));
  if (ti == tj) {                                      // below the diagonal: what is above it (E is symmetric)
    const int cc = lane & 31, rr = r & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r + i > c) out[i] = fmaf(fa, total((cc & 3) + 4 * (cc >> 3), rr + i + 32 * (cc >> 2 & 1)), fb * ev[i]);
  }
  store_planes4(j.C.hi, j.C.lo(), np, r, c, ti == tj, out);
}

// All products of a phase for np <= 128, one workgroup a matrix.  A wave owns one tile of 32 x 32 of every product (10 at
// np = 128).  Two matrices fit the LDS: A and P; S = A P and the next A are written over A, and the product Q of the steps
// is kept in its owners' registers and put where A was while it is multiplied.  The products are turns of ONE loop over the
// same few kilobytes of code.  Bound by instruction issue of the one CU: 3 waves a SIMD, each of which turns 16 results a
// lane into planes.
struct PhaseStage {
  int32_t what;                 // P: P = a I + b A + c A^2; S: A <- A P; A: A' = A P, held; Q: Q <- A P; W: no product
  int32_t out;                  // what is written over A behind it (P: over P): the result, the held A', Q
  int32_t first;                // P: it is Q too
  float alpha, beta, gamma;     // of the scaled values: result = alpha (L R) + beta A + gamma I
};
enum { ST_P, ST_S, ST_A, ST_Q, ST_W };
enum { OUT_RESULT, OUT_HELD, OUT_Q };
struct PhaseJob {
  Planes A, Q;
  int32_t n;
};
struct PhaseArgs {
  PhaseJob job[AGX_MAX_ORTH];
  PhaseStage stage[4 * PHASE + 1];
  int stages;
};
constexpr int PW = 10;          // waves of a phase's workgroup: the tiles of np = 128
constexpr int phase_lds(int np) { return 4 * np * (np + 8) * 2 + np / 32 * 32 * 33 * 4; }

template <int NP>
__device__ __forceinline__ void phase_steps(const PhaseArgs &a, const PhaseJob &j, _Float16 *A) {
  constexpr int nt = NP / 32, tri = nt * (nt + 1) / 2, LD = NP + 8, PL = NP * LD;   // (16 rows start in 16 bank groups)
  _Float16 *P = A + 2 * PL;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = (lane >> 5) * 8;
  for (int i = threadIdx.x * 8; i < NP * NP; i += PW * 64 * 8) {
    const int o = i / NP * LD + i % NP;
    *reinterpret_cast<half8 *>(&A[o]) = *reinterpret_cast<const half8 *>(j.A.hi + i);
    *reinterpret_cast<half8 *>(&A[PL + o]) = *reinterpret_cast<const half8 *>(j.A.lo() + i);
  }
  __syncthreads();
  int ti = 0, tj = 0;
  if (wave < tri) upper_tile(wave, nt, ti, tj);
  const bool diag = ti == tj;
  float *scratch = reinterpret_cast<float *>(A + 4 * PL) + ti * 32 * 33;
  const int c = tj * 32 + (lane & 31), r0 = ti * 32 + 4 * (lane >> 5);
  auto at = [](const _Float16 *p) { return *reinterpret_cast<const half8 *>(p); };
  float Q[16], held[16];
#pragma unroll 1
  for (int st = 0; st < a.stages; ++st) {
    const PhaseStage g = a.stage[st];
    float v[16];
    if (wave < tri && g.what != ST_W) {
      const _Float16 *l = A + (ti * 32 + (lane & 31)) * LD + h, *r = (g.what == ST_P ? A : P) + c * LD + h;
      f32x16 acc = {};
      // (the split's small terms are added first, so that only one product in three rounds at the sum's magnitude)
#pragma unroll
      for (int k = 0; k < NP; k += 64) {
        half8 x[4], y[4];
        f32x16 s = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = at(l + k + i * 16);
          y[i] = at(r + k + i * 16);
          s = __builtin_amdgcn_mfma_f32_32x32x16_f16(at(l + PL + k + i * 16), y[i], s, 0, 0, 0);
          s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i], at(r + PL + k + i * 16), s, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i], y[i], s, 0, 0, 0);
        acc += s;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = g.alpha * acc[i];
      if (g.what == ST_P) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {                  // (A is symmetric: its mirror image is one vector)
          const half4 eh = *reinterpret_cast<const half4 *>(&A[c * LD + r0 + 8 * q]), el = *reinterpret_cast<const half4 *>(&A[PL + c * LD + r0 + 8 * q]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[4 * q + i] += fmaf(g.beta, (float)eh[i] + (float)el[i], r0 + 8 * q + i == c && c < j.n ? g.gamma : 0.f);
        }
      }
      if (diag) {                                      // below the diagonal: what is above it (the wave's own 4 KB)
        const int lr = r0 & 31, lc = lane & 31;
#pragma unroll
        for (int i = 0; i < 16; ++i) scratch[(lr + 8 * (i >> 2) + (i & 3)) * 33 + lc] = v[i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = lr + 8 * (i >> 2) + (i & 3);
          const float m = scratch[lc * 33 + row];
          v[i] = row > lc ? m : v[i];
        }
      }
      if (g.first || g.what == ST_Q)
#pragma unroll
        for (int i = 0; i < 16; ++i) Q[i] = v[i];
      if (g.what == ST_A)
#pragma unroll
        for (int i = 0; i < 16; ++i) held[i] = v[i];
    }
    if (g.out == OUT_Q) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = Q[i];
    } else if (g.out == OUT_HELD) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = held[i];
    }
    __syncthreads();
    if (wave < tri) {
      _Float16 *o = g.what == ST_P ? P : A;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 w = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        store_planes4(o, o + PL, LD, r0 + 8 * q, c, diag, w);
      }
    }
    __syncthreads();
  }
  const _Float16 *f = a.stages == 1 ? P : A;           // (one step: P is the product)
  for (int i = threadIdx.x * 8; i < NP * NP; i += PW * 64 * 8) {
    const int o = i / NP * LD + i % NP;
    *reinterpret_cast<half8 *>(j.Q.hi + i) = *reinterpret_cast<const half8 *>(&f[o]);
    *reinterpret_cast<half8 *>(j.Q.lo() + i) = *reinterpret_cast<const half8 *>(&f[PL + o]);
  }
}
__global__ __launch_bounds__(PW * 64) void orth_phase_kernel(PhaseArgs a) {
  extern __shared__ _Float16 lds[];
  const PhaseJob &j = a.job[blockIdx.x];
  if (j.A.np == T) phase_steps<T>(a, j, lds);
  else phase_steps<2 * T>(a, j, lds);
}
static_assert(ONE_BLOCK == 2 * T, "one-workgroup phases are written for one or two tiles a side");

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
  int64_t maxb, invd, mat[5], part, trace, x[2], u, end;
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
  l.trace = take((int64_t)j.nt() * l.slices * 4);
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
      nb[i] = (int)std::min<int64_t>(MAXB, agx::cdiv64((int64_t)j.rows * agx::cdiv(j.cols, 4), 512));
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
  bool small = true;
  for (int i = 0; i < n; ++i) small = small && jobs[i].np() <= SMALL;
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
        g.trace = reinterpret_cast<float *>(base[i] + l.trace);
        g.first = gb;
        gb += tl * l.slices;
        ReduceJob &r = ra.job[i];
        r.part = g.part; r.trace = g.trace; r.maxb = g.maxb; r.invd = reinterpret_cast<double *>(base[i] + l.invd);
        r.A = planes(i, 0, exponent_for(s * s)); r.nt = nt; r.slices = l.slices; r.e = ex; r.nb = nb[i];
        r.normalise = first; r.first = rb;
        rb += tl * RCH;
      }
      hipLaunchKernelGGL(orth_gram_kernel, dim3(gb), dim3(256), 0, st, ga);
      AGX_LAUNCH_CHECK();
      hipLaunchKernelGGL(orth_reduce_kernel, dim3(rb), dim3(256), 0, st, ra);
      AGX_LAUNCH_CHECK();
    }
    // matrices: 0 A, 1 P, 2 A P, 3 / 4 Q (which of the two: 3 after an odd number of steps).  Matrices of np <= ONE_BLOCK take
    // the one-workgroup form, the others a launch per product
    const int steps = std::min(PHASE, o->steps - k);
    PhaseArgs pa;
    memset(&pa, 0, sizeof(pa));
    float coef[3 * PHASE];
    int eA[PHASE + 1], eP[PHASE], eS[PHASE], eQ[PHASE];              // scale exponents per step
    double bQ = 1.0;                                                 // |Q| <= bQ
    for (int t = 0; t < steps; ++t) {
      const float *c = o->coef + (o->n_coef == 1 ? 0 : 3 * (k + t));
      const Bounds b = bounds_of(s, c[0], c[1], c[2]);
      memcpy(coef + 3 * t, c, 3 * sizeof(float));
      bQ *= b.P;
      eA[t] = exponent_for(s * s); eP[t] = exponent_for(b.P); eS[t] = exponent_for(b.S); eQ[t] = exponent_for(bQ);
      s = b.next;
    }
    eA[steps] = exponent_for(s * s);
    k += steps;
    const int iq = steps & 1 ? 3 : 4;
    for (int t = 0; t < steps; ++t) {
      const bool more = t + 1 < steps;
      auto stage = [&](int what, int e, int out) -> PhaseStage & {
        PhaseStage &g = pa.stage[pa.stages++];
        g.what = what; g.alpha = std::ldexp(1.f, e); g.out = out;
        return g;
      };
      PhaseStage &p = stage(ST_P, 0, OUT_RESULT);
      p.alpha = std::ldexp(coef[3 * t + 2], eP[t] - 2 * eA[t]);
      p.beta = std::ldexp(coef[3 * t + 1], eP[t] - eA[t]);
      p.gamma = std::ldexp(coef[3 * t], eP[t]);
      p.first = t == 0;
      if (more) stage(ST_S, eS[t] - eA[t] - eP[t], OUT_RESULT);
      if (more) stage(ST_A, eA[t + 1] - eS[t] - eP[t], t > 0 ? OUT_Q : OUT_RESULT);
      if (t > 0 && !more) stage(ST_W, 0, OUT_Q);
      if (t > 0) stage(ST_Q, eQ[t] - eQ[t - 1] - eP[t], more ? OUT_HELD : OUT_Q);
    }
    int nblock = 0, lds = 0;
    for (int i = 0; i < n; ++i)
      if (jobs[i].np() <= ONE_BLOCK) {
        PhaseJob &g = pa.job[nblock++];
        g.A = planes(i, 0, 0); g.Q = planes(i, iq, 0); g.n = jobs[i].n();
        lds = std::max(lds, phase_lds(jobs[i].np()));
      }
    if (nblock) {
      hipLaunchKernelGGL(orth_phase_kernel, dim3(nblock), dim3(PW * 64), lds, st, pa);
      AGX_LAUNCH_CHECK();
    }
    for (int t = 0; t < steps && nblock < n; ++t) {
      const int in = t & 1 ? 3 : 4, out = t & 1 ? 4 : 3, iP = t == 0 ? out : 1;   // the first step's P is Q too
      auto launch = [&](int per, auto fill) -> int {
        ChainArgs ca;
        int blocks = 0;
        ca.n = 0;
        for (int i = 0; i < n; ++i)
          for (int w = 0; w < per && jobs[i].np() > ONE_BLOCK; ++w) {
            ChainJob &g = ca.job[ca.n++];
            memset(&g, 0, sizeof(g));
            g.n = jobs[i].n(); g.nt = small ? jobs[i].np() / 32 : jobs[i].nt(); g.first = blocks; g.alpha = 1.f;
            blocks += g.nt * (g.nt + 1) / 2;
            fill(g, i, w);
          }
        if (small) hipLaunchKernelGGL(orth_chain_small_kernel, dim3(blocks), dim3(256), 0, st, ca);
        else hipLaunchKernelGGL(orth_chain_kernel, dim3(blocks), dim3(256), 0, st, ca);
        AGX_LAUNCH_CHECK();
        return AGX_OK;
      };
      AGX_TRY(launch(1, [&](ChainJob &g, int i, int) {               // P = a I + b A + c A^2
        g.L = g.R = g.E = planes(i, 0, eA[t]);
        g.C = planes(i, iP, eP[t]);
        g.alpha = coef[3 * t + 2]; g.beta = coef[3 * t + 1]; g.gamma = coef[3 * t];
      }));
      const bool more = t + 1 < steps;
      const int two = (more ? 1 : 0) + (t > 0 ? 1 : 0);
      if (two)
        AGX_TRY(launch(two, [&](ChainJob &g, int i, int w) {         // S = A P (where a step follows) | Q <- Q P
          const bool sp = more && w == 0;
          g.R = planes(i, iP, eP[t]);
          g.L = sp ? planes(i, 0, eA[t]) : planes(i, in, eQ[t > 0 ? t - 1 : 0]);
          g.C = sp ? planes(i, 2, eS[t]) : planes(i, out, eQ[t]);
        }));
      if (more)
        AGX_TRY(launch(1, [&](ChainJob &g, int i, int) {             // A <- S P
          g.L = planes(i, 2, eS[t]);
          g.R = planes(i, iP, eP[t]);
          g.C = planes(i, 0, eA[t + 1]);
        }));
    }
    ApplyArgs aa;
    aa.n = n;
    int blocks = 0;
    for (int i = 0; i < n; ++i) {
      const Job &j = jobs[i];
      ApplyJob &g = aa.job[i];
      memset(&g, 0, sizeof(g));
      g.x = x[i]; g.ldx = ldx[i]; g.Q = planes(i, iq, eQ[steps - 1]);
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
    AGX_CHECK_ARG((int64_t)a.rows * agx::cdiv64(a.cols, 4) < (1LL << 30) && agx::cdiv64(a.rows, T) * agx::cdiv64(a.cols, T) < (1 << 26),
                  "%s: matrix %d is too large", who, i);
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

// (a phase in one workgroup takes more LDS than the default limit of a launch)
int agx::orth_prepare_device() {
  AGX_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&orth_phase_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              phase_lds(ONE_BLOCK)));
  return AGX_OK;
}

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
