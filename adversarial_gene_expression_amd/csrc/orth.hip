// Orthogonalised updates: Newton-Schulz steps X <- X (a I + b A + c A^2), A = X^T X, on matrices whose smaller side n is
// far below the larger one (a Dense kernel over genes: 18161 x 256).
//
// Algebra.  All iterates are X_0 times polynomials of A_0, which commute, so several steps need the long side only twice:
// with P = aI + bA + cA^2 the next Gram matrix is A P^2 and the product of the steps Q <- Q P; X_k = X_0 Q.  An error of
// A_0 in a direction of tiny singular value grows with every step (by up to a^2 in A), so two or three steps are taken this
// way (phase_of); then X Q is formed and its Gram matrix computed anew.
// Matrices of n x n are symmetric: tiles on and above the diagonal are computed and mirrored.
//
// Products run on the fp16 matrix cores: every operand is split into two fp16 terms, v 2^e = hi + lo (22 bits where fp32 has
// 24), and hi.hi + hi.lo + lo.hi are accumulated in fp32 (lo.lo is below 2^-22 of the product).  e is one for a matrix: from the
// largest |x| for the caller's (first launch), from a bound on the spectral norm, worked out on the host, for everything
// behind it.  Entries then stay under 2^14, the largest (or the bound) at 2^13 or more; fp16's last bit is 2^-24, so that an
// entry down to 2^-16 of the largest keeps its 22 bits and any is off by at most 2^-38 of the largest: rows or columns
// that are far smaller than the others come out less exactly than in fp32 (a block at 1e-5 of the rest to 2e-6, at 1e-6 to 2e-5).  A bf16
// operand needs one term only: its 8 bits fit, down to the same 2^-38.
//
// Launches of a call: the momentum step with |x|'s maximum and norm; then, a phase each, the Gram matrix (and the sum of its
// slices), its polynomial (n <= 128 one launch a phase, n <= 256 one a step, above three a step) and the product with the
// long side, which in the last phase is the Muon update of w too.  Floors: 2.4 us a launch, 5 TB/s of HBM, 1150 TFLOP/s of
// fp16 products over three.  Measured: 256 x 256 88 us (12 launches), 18161 x 256 147 us (15), 1000 x 4297 bf16 360 us
// (19; its products take 73 us at that rate).
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

constexpr int T = 64;                          // n x n matrices are padded to T, 2 T, 4 T or a multiple of T above
constexpr int PHASE = 3;                       // most steps between two Gram matrices
constexpr int MAXB = 1024;                     // workgroups of a matrix's first launch, each with its share of maximum and squares
constexpr int ROWS_PHASE = 128;                // largest padded side for a phase in one launch
constexpr int TALL_BLOCKS = 2, WIDE_BLOCKS = 4;    // workgroups a CU of a Gram product
constexpr int ONE_SLICE = 4;                   // longest K, in steps of 64 (1.5 us each), that is not split over workgroups
constexpr int LINES_BLOCKS = 2, ONE_SLICE_LINES = 16;   // the same of the iterate's Gram product (see run)
constexpr int FEW_SLICES = 16;                 // see orth_reduce_kernel
constexpr int TARGET = 14;                     // scaled entries are below 2^TARGET

// n x n matrix as two fp16 planes of np x np (np: n rounded up, zeros behind), value = (hi + lo) 2^-e, in the order of the
// matrix cores' operands, so that a wave's load of 16 rows and 32 k is one piece of 1 KB: blocks of 16 rows by 64 k, in them
// (k / 8) % 2, then (k / 16) % 4, the row and k % 8.  (Row-major, each of those loads asks for 16 bytes of 32 lines or more.)
struct Planes {
  _Float16 *hi;
  int32_t e, np;
  __device__ __forceinline__ _Float16 *lo() const { return hi + (int64_t)np * np; }
};
constexpr int NEXT_ROW = 8;                    // from a place to the same k of the next row, inside a block
__device__ __forceinline__ int place(int np, int row, int k) {        // (eight k's from a multiple of 8 on are neighbours)
  return (((row >> 4) * (np >> 6) + (k >> 6)) * 2 + ((k >> 3) & 1)) * 512 + (((k >> 4) & 3) * 16 + (row & 15)) * 8 + (k & 7);
}
__device__ __forceinline__ void placed(int np, int piece, int &row, int &k) {   // of the piece-th eight values in operand order
  const int block = piece >> 7;
  row = block / (np >> 6) * 16 + (piece & 15);
  k = block % (np >> 6) * 64 + (piece >> 4 & 3) * 16 + (piece >> 6 & 1) * 8;
}

__device__ __forceinline__ int exponent_of(uint32_t absbits) {   // e with |v| < 2^e for the float of these bits
  return absbits == 0 ? 0 : (int)(absbits >> 23) - 126;
}
// The iterate between two phases: its K lines (rows of a tall matrix, columns of a wide one) of n values as planes of np rows
// by kp lines (K rounded up to 64; zeros behind n and K), in the same order: the operands of its Gram matrix.
struct Lines {
  _Float16 *hi;
  int64_t kp;
  int32_t e, np;
  __device__ __forceinline__ _Float16 *lo() const { return hi + np * kp; }
  __device__ __forceinline__ int64_t at(int i, int line) const {     // value i of a line (eight lines are neighbours)
    return ((i >> 4) * (kp >> 6) + (line >> 6)) * 1024 + ((line >> 3) & 1) * 512 + (((line >> 4) & 3) * 16 + (i & 15)) * 8 + (line & 7);
  }
};

// v = hi + lo, each rounded to nearest (two values an instruction)
__device__ __forceinline__ void split4(f32x4 v, half4 &hi, half4 &lo) {
  hi = __builtin_convertvector(v, half4);
  lo = __builtin_convertvector(v - __builtin_convertvector(hi, f32x4), half4);
}

// ---------------------------------------------------------------------------------------------------------------------
// largest |x| and sum of squares; with a momentum step in front where m is given: m <- mu m + g, u = g + mu m (nesterov) or m
// ---------------------------------------------------------------------------------------------------------------------
struct PrepJob {
  const void *x;        // matrix (g with momentum)
  float *m, *u;         // momentum buffer; where u goes (NULL: u is m)
  int64_t ldx, ldm, ldu;
  int32_t rows, cols, dtype, nb;
  uint32_t *maxb;       // a workgroup's share of each
  double *squares;
};
struct PrepArgs {
  PrepJob job[AGX_MAX_ORTH];
  float mu;
  int nesterov;
};

template <typename E> struct Vec4;
template <> struct Vec4<float> { typedef f32x4u type; };
template <> struct Vec4<__bf16> { typedef bf16x4u type; };
// four values at p, zeros from the n-th on
template <typename E>
__device__ __forceinline__ f32x4 load4z(const E *p, int n) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (n >= 4) {
    const typename Vec4<E>::type w = *reinterpret_cast<const typename Vec4<E>::type *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < n) v[i] = (float)p[i];
  }
  return v;
}
__device__ __forceinline__ void store4(float *p, int n, f32x4 v) {
  if (n >= 4) {
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
  __shared__ double sums[4];
  uint32_t mx = 0;
  double sq = 0.0;
  const uint32_t per_row = (uint32_t)(j.cols + 3) / 4;               // (host: rows * per_row < 2^31)
  const uint32_t items = per_row * (uint32_t)j.rows, step = (uint32_t)j.nb * 256;
#pragma unroll 4
  for (uint32_t it = blockIdx.x * 256 + threadIdx.x; it < items; it += step) {
    const uint32_t r = it / per_row;
    const int c = (int)(it - r * per_row) * 4, n = min(4, j.cols - c);
    f32x4 v = j.dtype == AGX_F32 ? load4z(reinterpret_cast<const float *>(j.x) + (int64_t)r * j.ldx + c, n)
                                 : load4z(reinterpret_cast<const __bf16 *>(j.x) + (int64_t)r * j.ldx + c, n);
    if (j.m) {
      f32x4 m = load4z(j.m + (int64_t)r * j.ldm + c, n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = a.mu * m[i] + v[i];
        v[i] = a.nesterov ? v[i] + a.mu * m[i] : m[i];
      }
      store4(j.m + (int64_t)r * j.ldm + c, n, m);
      if (j.u) store4(j.u + (int64_t)r * j.ldu + c, n, v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);              // (as integers: infinities and NaN win)
      sq = fma((double)v[i], (double)v[i], sq);                        // (64 bits: no overflow or underflow to look after)
    }
  }
  sq = agx::wave_sum(sq);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = mx;
    sums[threadIdx.x >> 6] = sq;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    j.maxb[blockIdx.x] = max(max(red[0], red[1]), max(red[2], red[3]));
    j.squares[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}

// tile (ti <= tj) of linear index t over the upper triangle of nt x nt tiles (nt is small: no square root)
__device__ __forceinline__ void upper_tile(int t, int nt, int &ti, int &tj) {
  ti = 0;
  while (t >= nt - ti) t -= nt - ti++;
  tj = ti + t;
}

// scale exponent of a matrix from its partial maxima; every thread of the workgroup gets it (red: a word a wave)
__device__ __forceinline__ int scale_exponent(const uint32_t *maxb, int nb, uint32_t *red) {
  uint32_t mx = 0;
  for (int i = threadIdx.x; i < nb; i += blockDim.x) mx = max(mx, maxb[i]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
  __syncthreads();
  mx = 0;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) mx = max(mx, red[i]);
  return TARGET - exponent_of(mx);
}

// 1 / (|X|_F + eps) of the matrix scaled by 2^e, the same in every thread and workgroup (sums: a word a wave).  A matrix of
// zeros gives zeros, one with an infinity or NaN NaN throughout.
__device__ __forceinline__ double normaliser(const double *squares, int nb, float eps, int e, double *sums) {
  double s = 0.0;
  for (int i = threadIdx.x; i < nb; i += blockDim.x) s += squares[i];
  s = agx::wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) s += sums[i];
  if (!(s < __builtin_huge_val())) return __builtin_nan("");
  return s == 0.0 ? 0.0 : 1.0 / ldexp(sqrt(s) + (double)eps, e);
}

// ---------------------------------------------------------------------------------------------------------------------
// tile product: operands in LDS as [64 rows][64 k] fp16 planes (the first Gram product, and for n > 256 the product with the
// long side).  K in steps of 64 through one buffer, the next step's global loads in flight: four workgroups of a CU overlap
// each other's loads, conversions and products.  (Two or four steps in flight: fewer workgroups, 18161 x 256 157 us became
// 172; tiles of 128 x 128 with two buffers leave one workgroup a CU, whose phases nothing covers: 166 where this took 158.)
// ---------------------------------------------------------------------------------------------------------------------
constexpr int BK = 64, LDK = BK + 8, PL = T * LDK;   // k of a step; LDS rows of 144 bytes (16 of them start in 16 different bank
                                                     // groups); halves of a plane
__device__ __forceinline__ f32x4 scale4(f32x4 v, int e) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_ldexpf(v[i], e);
  return v;
}

// The loaders keep one 64-bit base a tile, the same for all lanes, and 32-bit offsets of their own (the host checks that 128
// rows of a leading dimension fit them).
// rows r0.. of a planes matrix, k contiguous (a symmetric matrix: also its columns)
struct LoadPlanes {
  static constexpr bool two = true;
  const _Float16 *hi, *lo;
  int np;
  half8 v[4];
  __device__ __forceinline__ explicit LoadPlanes(const Planes &m) : hi(m.hi), lo(m.lo()), np(m.np) {}
  __device__ __forceinline__ void fetch(int64_t r0, int64_t k0) {
    const _Float16 *bh = hi + r0 * np + k0 * 16, *bl = lo + r0 * np + k0 * 16;      // (block (r0, k0) of 16 x 64)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int o = ((threadIdx.x >> 7) + 2 * p) * 16 * np + (threadIdx.x & 127) * 8;
      v[2 * p] = *reinterpret_cast<const half8 *>(bh + o);
      v[2 * p + 1] = *reinterpret_cast<const half8 *>(bl + o);
    }
  }
  __device__ __forceinline__ void store(_Float16 *t) const {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      int row, k;
      placed(BK, threadIdx.x + 256 * p, row, k);
      const int o = row * LDK + k;
      *reinterpret_cast<half8 *>(t + o) = v[2 * p];
      *reinterpret_cast<half8 *>(t + PL + o) = v[2 * p + 1];
    }
  }
};

// (raw vectors are kept until they are stored: a conversion would wait for the load.  Tiles inside the matrix, which are
// nearly all, take plain loads; at its edges every element is looked at.)
// rows r0.. of a caller's matrix, k contiguous; zeros outside [rows) x [kmax)
template <typename E> struct LoadK {
  static constexpr bool two = sizeof(E) == 4;
  using V = typename Vec4<E>::type;
  const E *p;
  int64_t ld, rows, kmax;
  int e;
  V v[4];
  __device__ __forceinline__ void fetch(int64_t r0, int64_t k0) {
    const E *b = p + r0 * ld + k0;
    const int row = threadIdx.x >> 4, k = (threadIdx.x & 15) * 4;
    if (r0 + T <= rows && k0 + BK <= kmax) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const V *>(b + (row + 16 * q) * (int)ld + k);
    } else {
      const int nk = (int)min((int64_t)BK, kmax - k0) - k, nr = (int)min((int64_t)T, rows - r0);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[q][i] = row + 16 * q < nr && i < nk ? b[(row + 16 * q) * (int)ld + k + i] : (E)0.f;
    }
  }
  __device__ __forceinline__ void store(_Float16 *t) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int o = ((threadIdx.x >> 4) + 16 * q) * LDK + (threadIdx.x & 15) * 4;
      const V w = v[q];
      half4 hi, lo;
      split4(scale4(f32x4{(float)w[0], (float)w[1], (float)w[2], (float)w[3]}, e), hi, lo);
      *reinterpret_cast<half4 *>(t + o) = hi;
      if (two) *reinterpret_cast<half4 *>(t + PL + o) = lo;
    }
  }
};

// columns r0.. of a caller's matrix whose rows are k: element (r, k) at p[k * ld + r].  A thread takes a block of 4 x 4: four
// k's of four columns, so that loads and LDS writes are both vectors; a wave covers 32 columns of 32 k's (64 bytes or more
// of a row, and LDS writes without bank conflicts).
template <typename E> struct LoadT {
  static constexpr bool two = sizeof(E) == 4;
  using V = typename Vec4<E>::type;
  const E *p;
  int64_t ld, rows, kmax;
  int e;
  V v[4];                                              // v[k][column]
  __device__ __forceinline__ int col() const { return (threadIdx.x >> 7) * 32 + (threadIdx.x & 7) * 4; }
  __device__ __forceinline__ int kk() const { return (threadIdx.x >> 3 & 15) * 4; }
  __device__ __forceinline__ void fetch(int64_t r0, int64_t k0) {
    const E *b = p + k0 * ld + r0;
    const int c = col(), k = kk();
    if (r0 + T <= rows && k0 + BK <= kmax) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const V *>(b + (k + i) * (int)ld + c);
    } else {
      const int nr = (int)min((int64_t)T, rows - r0) - c, nk = (int)min((int64_t)BK, kmax - k0);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[i][q] = k + i < nk && q < nr ? b[(k + i) * (int)ld + c + q] : (E)0.f;
    }
  }
  __device__ __forceinline__ void store(_Float16 *t) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int o = (col() + i) * LDK + kk();
      half4 hi, lo;
      split4(scale4(f32x4{(float)v[0][i], (float)v[1][i], (float)v[2][i], (float)v[3][i]}, e), hi, lo);
      *reinterpret_cast<half4 *>(t + o) = hi;
      if (two) *reinterpret_cast<half4 *>(t + PL + o) = lo;
    }
  }
};

// lines r0.. of the iterate, k the values of a line; blocks of 4 x 4 as above
struct LoadLines {
  static constexpr bool two = true;
  const Lines *x;
  int e;                                               // (not used: the planes are scaled)
  half4 vh[4], vl[4];                                  // [k][line]
  __device__ __forceinline__ int line() const { return (threadIdx.x >> 7) * 32 + (threadIdx.x & 7) * 4; }
  __device__ __forceinline__ int kk() const { return (threadIdx.x >> 3 & 15) * 4; }
  __device__ __forceinline__ void fetch(int64_t r0, int64_t k0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t o = x->at((int)k0 + kk() + i, (int)r0 + line());
      vh[i] = *reinterpret_cast<const half4 *>(x->hi + o);
      vl[i] = *reinterpret_cast<const half4 *>(x->lo() + o);
    }
  }
  __device__ __forceinline__ void store(_Float16 *t) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int o = (line() + i) * LDK + kk();
      *reinterpret_cast<half4 *>(t + o) = half4{vh[0][i], vh[1][i], vh[2][i], vh[3][i]};
      *reinterpret_cast<half4 *>(t + PL + o) = half4{vl[0][i], vl[1][i], vl[2][i], vl[3][i]};
    }
  }
};

// acc = A-tile (rows ra..) . B-tile (rows rb..)^T over k in [k0, k1), whole steps.  The matrix cores add a step's products,
// the split's small terms first, and vector additions the steps: a long chain of additions to one fp32 sum would lose what
// the split keeps.  same: both operands are the same rows, loaded once.
// late(): called when the first loads are on their way (sets the scale exponents the stores use).
template <class LA, class LB, class Late>
__device__ __forceinline__ f32x16 tile_product(LA &la, LB &lb, int64_t ra, int64_t rb, int64_t k0, int64_t k1, _Float16 *lds,
                                               bool same, Late late) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fa = ((wave >> 1) * 32 + (lane & 31)) * LDK + (lane >> 5) * 8;
  const int fb = ((wave & 1) * 32 + (lane & 31)) * LDK + (lane >> 5) * 8 + (same ? 0 : 2 * PL);
  f32x16 acc = {};
  auto fetch = [&](int64_t k) {
    la.fetch(ra, k);
    if (!same) lb.fetch(rb, k);
  };
  auto at = [&](int o) { return *reinterpret_cast<const half8 *>(lds + o); };
  fetch(k0);
  late();
  for (int64_t k = k0; k < k1; k += BK) {
    la.store(lds);
    if (!same) lb.store(lds + 2 * PL);
    if (k + BK < k1) fetch(k + BK);
    __syncthreads();
    f32x16 sum = {};
#pragma unroll
    for (int i = 0; i < BK; i += 32) {
      const half8 a0 = at(fa + i), a1 = at(fa + i + 16), b0 = at(fb + i), b1 = at(fb + i + 16);
      if constexpr (LA::two) {
        sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(at(PL + fa + i), b0, sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(at(PL + fa + i + 16), b1, sum, 0, 0, 0);
      }
      if constexpr (LB::two) {
        sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, at(PL + fb + i), sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(a1, at(PL + fb + i + 16), sum, 0, 0, 0);
      }
      sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, b0, sum, 0, 0, 0);
      sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(a1, b1, sum, 0, 0, 0);
    }
    acc += sum;
    __syncthreads();
  }
  return acc;
}
// calls f(row, column, value) for a lane's elements of the tile
template <class Fn>
__device__ __forceinline__ void each_element(const f32x16 &acc, Fn f) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int e = 0; e < 16; ++e) f((wave >> 1) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), (wave & 1) * 32 + (lane & 31), acc[e]);
}

// ---------------------------------------------------------------------------------------------------------------------
// Gram matrix of the caller's matrix, K split over workgroups: partial tiles [tile][slice][64][64] of the scaled matrix
// ---------------------------------------------------------------------------------------------------------------------
struct GramJob {
  const void *x;
  int64_t ld, K, kper;          // K: long side; kper: k of one slice (a multiple of BK)
  int32_t n, nt, slices, tall;  // n: small side, nt: tiles along it; tall: element (i, k) at x[k * ld + i]
  int32_t dtype, nb;            // nb: shares of the maximum (the scale's) and of the sum of squares
  const uint32_t *maxb;
  float *part;
  const double *squares;        // this, invd and A: for one slice, as in ReduceJob
  double *invd;
  Planes A;
  int32_t first;                // first workgroup of the job
};
struct GramArgs {
  GramJob job[AGX_MAX_ORTH];
  int n;
  float eps;
};

template <class L>
__device__ __forceinline__ f32x16 gram_tile(const GramJob &j, int ti, int tj, int64_t k0, int64_t k1, int &e, uint32_t *red, _Float16 *lds) {
  L la, lb;
  la.p = reinterpret_cast<decltype(la.p)>(j.x);
  la.ld = j.ld; la.rows = j.n; la.kmax = j.K;
  lb.p = la.p; lb.ld = la.ld; lb.rows = la.rows; lb.kmax = la.kmax;
  return tile_product(la, lb, (int64_t)ti * T, (int64_t)tj * T, k0, k1, lds, ti == tj,
                      [&] { la.e = lb.e = e = scale_exponent(j.maxb, j.nb, red); });
}

// Symmetric results are made symmetric to the last bit, from what is on and above the diagonal: products of matrices that are
// symmetric up to rounding are not, and the iteration would multiply the difference (rank-deficient matrices: 50 times the
// error).
// A lane's four rows r.. of column c go out as pairs of columns, which two neighbouring lanes exchange (the even one takes the
// first two rows, the odd one the others)
__device__ __forceinline__ void store_pairs4(_Float16 *p, int ld, int r, int c, half4 x) {
  const bool odd = threadIdx.x & 1;
  const uint2 w = __builtin_bit_cast(uint2, x);        // rows (0, 1) and (2, 3) of this lane's column
  const uint32_t mine = odd ? w.y : w.x, give = odd ? w.x : w.y;
  const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0xb1, 0xf, 0xf, true);   // lanes 2 k <-> 2 k + 1
  const uint32_t a = odd ? got : mine, b = odd ? mine : got;
  uint32_t *q = reinterpret_cast<uint32_t *>(p + (r + (odd ? 2 : 0)) * ld + (c & ~1));
  q[0] = (a & 0xffffu) | (b << 16);
  *reinterpret_cast<uint32_t *>(reinterpret_cast<_Float16 *>(q) + ld) = (a >> 16) | (b & 0xffff0000u);
}
// The same of a symmetric matrix, into planes with their mirror image, which is contiguous.  diag: the tile's mirror image is
// all of it.
__device__ __forceinline__ void store_planes4(const Planes &m, int r, int c, bool diag, f32x4 v) {
  half4 h, l;
  split4(v, h, l);
  const int o = place(m.np, c, r), x = place(m.np, r, c & ~1);
  *reinterpret_cast<half4 *>(m.hi + o) = h;
  *reinterpret_cast<half4 *>(m.lo() + o) = l;
  if (diag) return;                                    // (uniform over the wave)
  store_pairs4(m.hi + x, NEXT_ROW, 0, 0, h);
  store_pairs4(m.lo() + x, NEXT_ROW, 0, 0, l);
}
// A lane's results of a 32 x 32 tile on the diagonal (rows lr + 8 (i / 4) + i % 4 of column lc): what is below it from what
// is above, through 32 * 33 words of the wave's own
__device__ __forceinline__ void mirror(float *v, float *scratch) {
  const int lane = threadIdx.x & 63, lr = 4 * (lane >> 5), lc = lane & 31;
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

// KIND: what all of a launch's matrices are (bit 0: wide, bit 1: bf16), or ANY: one loader's registers instead of the
// largest of four let twice as many workgroups of a CU wait for memory at a time
constexpr int ANY = 4, ITERATE = 5;            // (ITERATE: the planes between two phases)
__device__ __host__ __forceinline__ bool is_kind(int kind, bool tall, int dtype) { return kind == (tall ? 0 : 1) + (dtype == AGX_F32 ? 0 : 2); }

// ONE: the job is one slice, and its tiles (of all np x np) go out as A_0 itself, without a launch that adds slices
template <int KIND, bool ONE>
__global__ __launch_bounds__(256, 4) void orth_gram_kernel(GramArgs a) {
  __shared__ __align__(16) _Float16 lds[4 * PL];
  __shared__ uint32_t red[4];
  // (the tiles of one slice follow each other on one XCD, whose L2 then reads the slice once)
  const int id = agx::xcd_logical_id(blockIdx.x, gridDim.x);
  int q = 0;
  while (q + 1 < a.n && id >= a.job[q + 1].first) ++q;
  const GramJob &j = a.job[q];
  const int tiles = j.nt * (j.nt + 1) / 2, slice = ONE ? 0 : (id - j.first) / tiles, tile = (id - j.first) % tiles;
  int ti, tj, e;
  upper_tile(tile, j.nt, ti, tj);
  const int64_t k0 = (int64_t)slice * j.kper, k1 = min(k0 + j.kper, (j.K + BK - 1) / BK * BK);
  f32x16 acc;
  auto is = [&](int kind) { return KIND == ANY ? is_kind(kind, j.tall, j.dtype) : KIND == kind; };
  if (is(0)) acc = gram_tile<LoadT<float>>(j, ti, tj, k0, k1, e, red, lds);
  else if (is(1)) acc = gram_tile<LoadK<float>>(j, ti, tj, k0, k1, e, red, lds);
  else if (is(2)) acc = gram_tile<LoadT<__bf16>>(j, ti, tj, k0, k1, e, red, lds);
  else acc = gram_tile<LoadK<__bf16>>(j, ti, tj, k0, k1, e, red, lds);
  if constexpr (!ONE) {
    float *p = j.part + ((int64_t)tile * j.slices + slice) * T * T;
    each_element(acc, [&](int r, int c, float v) { p[r * T + c] = v; });
  } else {
    __shared__ double sums[4];
    const double inv = normaliser(j.squares, j.nb, a.eps, e, sums), f = ldexp(inv * inv, j.A.e);
    if (tile == 0 && threadIdx.x == 0) *j.invd = inv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fi = 2 * ti + (wave >> 1), fj = 2 * tj + (wave & 1);
    if (fi > fj) return;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = (float)((double)acc[i] * f);
    if (fi == fj) mirror(v, reinterpret_cast<float *>(lds) + wave * 32 * 33);
#pragma unroll
    for (int p = 0; p < 4; ++p)
      store_planes4(j.A, fi * 32 + 4 * (lane >> 5) + 8 * p, fj * 32 + (lane & 31), fi == fj, f32x4{v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]});
  }
}

// A_0 = (sum of the partial Gram tiles) / d^2 with d = |X|_F + eps (first phase) or without a divisor (later phases).
// A workgroup takes R rows of a square of 32 x 32 on or above the diagonal: interleaved shares of the slices meet in LDS, from
// where the piece and its mirror image go out as vectors.  R = 32 (4 shares) where the slices are few, 4 (8 shares) where
// they are many: 18161 x 256 (48 slices) 5.6 us instead of 7.1, 4318 x 128 5.4 instead of 6.8; 1000 x 4297 (7 slices) 13.7 us
// instead of 17.4, 640 x 2000 6.5 instead of 7.4.
struct ReduceJob {
  const float *part;
  const uint32_t *maxb;
  const double *squares;
  double *invd;                 // 1 / d of the scaled matrix, for the product with the long side (phase 0)
  Planes A;
  int32_t nt, slices, e, nb, normalise, first;         // nt: partial tiles along a side
};
struct ReduceArgs {
  ReduceJob job[AGX_MAX_ORTH];
  int n;
  float eps;
};
template <int R> constexpr int reduce_threads() { return R == 32 ? 1024 : 256; }
template <int R>
__global__ __launch_bounds__(reduce_threads<R>()) void orth_reduce_kernel(ReduceArgs a) {
  constexpr int NT = reduce_threads<R>(), NG = NT / (R * 8);   // shares
  __shared__ float piece[NG][R][33];
  __shared__ uint32_t red[16];
  __shared__ double tr[16];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const ReduceJob &j = a.job[q];
  int pi, pj;                                          // square of the n x n matrix, and where it is in the partial tiles
  upper_tile((blockIdx.x - j.first) / (32 / R), j.A.np / 32, pi, pj);
  const int r0 = (blockIdx.x - j.first) % (32 / R) * R;
  constexpr int per = T / 32, area = T * T;
  const int ti = pi / per, tj = pj / per;
  const int tile = ti * j.nt - ti * (ti - 1) / 2 + tj - ti;
  const int grp = threadIdx.x / (R * 8), r = (threadIdx.x >> 3) % R, c = (threadIdx.x & 7) * 4;
  const float *p = j.part + (int64_t)tile * j.slices * area + (pi % per * 32 + r0 + r) * T + pj % per * 32 + c;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int z = grp; z < (tj < j.nt ? j.slices : 0); z += NG) sum += *reinterpret_cast<const f32x4 *>(p + (int64_t)z * area);
#pragma unroll
  for (int i = 0; i < 4; ++i) piece[grp][r][c + i] = sum[i];
  double f;
  if (j.normalise) {
    const int e = scale_exponent(j.maxb, j.nb, red);
    const double inv = normaliser(j.squares, j.nb, a.eps, e, tr);
    f = ldexp(inv * inv, j.A.e);
    if ((int)blockIdx.x == j.first && threadIdx.x == 0) *j.invd = inv;
  } else {
    f = ldexp(1.0, j.A.e - 2 * j.e);
  }
  __syncthreads();
  auto total = [&](int y, int x) {
    float t = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) t += piece[g][y][x];
    return (float)((double)t * f);
  };
  // the first threads write the piece, the next its mirror image
  const int y0 = pi * 32 + r0, x0 = pj * 32, np = j.A.np;
  f32x4 v;
  half4 h, l;
  int row, col;
  if (grp == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = total(r, c + i);
    row = y0 + r;
    col = x0 + c;
  } else if (grp == 1) {                               // (32 rows of R columns)
    const int x = threadIdx.x % (R * 8) / (R / 4), y = threadIdx.x % (R / 4) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = total(y + i, x);
    row = x0 + x;
    col = y0 + y;
  } else {
    return;
  }
  split4(v, h, l);
  const int o = place(np, row, col);
  if (pi != pj) {
    *reinterpret_cast<half4 *>(j.A.hi + o) = h;
    *reinterpret_cast<half4 *>(j.A.lo() + o) = l;
  } else {                                             // what is on and above the diagonal, and its mirror image
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (grp == 0 ? row <= col + i : row > col + i) {
        j.A.hi[o + i] = h[i];
        j.A.lo()[o + i] = l[i];
      }
    }
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

// A workgroup has a tile of 64 x 32 on or above the diagonal, its four waves every fourth step of 64 k of all of it: operands
// go straight from L2 to the matrix cores' registers, each byte once a workgroup, without LDS or barriers until the waves'
// sums meet.  (Tiles through LDS, four or eight waves at a barrier a step: 16.5 us at n = 1024 instead of 15.1, 12.5 at 640
// instead of 8.2.)  At n = 1024, 14 us a launch: the matrix cores work 1.5 us in the mean, a wave lives 8 us and waits for 30% of
// it (186 registers and 272 tiles on 256 CUs: mostly one wave a SIMD), a CU with two tiles reads 786 KB or 5.1 us at 64 bytes a
// clock, a quarter of the L2s' requests miss (13.6 MB from the last-level cache), the launch is 2.4.  No one of them bounds it.
typedef float WaveSums[4][32][64];                    // [wave][element of two accumulators][lane]
// tile of 64 x 32 of linear index t: row ti of tiles starts at column 2 ti
__device__ __forceinline__ void half_tile(int t, int nt, int &ti, int &tj) {
  ti = 0;
  while (t >= 2 * (nt - ti)) t -= 2 * (nt - ti++);
  tj = t + 2 * ti;
}
// the workgroup's product of 64 rows (x) and 32 rows (y) over steps s0.. < s1 of 64 k into `part`; rs: values of 16 rows
__device__ __forceinline__ void wave_products(const _Float16 *xh, const _Float16 *xl, const _Float16 *yh, const _Float16 *yl, int64_t rs,
                                              int s0, int s1, WaveSums &part) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (k runs in an order of its own, the same for both operands)
  const int64_t at = (lane & 31) / 16 * rs + (lane >> 5) * 128 + (lane & 15) * 8;
  half8 x[2][2][2][2], y[2][2][2];                     // [half of a step][rows 32 ..][plane][vector], [half][plane][vector]
  auto fetch = [&](int s, int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t o = at + (int64_t)s * 1024 + h * 256 + i * 512;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        x[h][t][0][i] = *reinterpret_cast<const half8 *>(xh + t * 2 * rs + o);
        x[h][t][1][i] = *reinterpret_cast<const half8 *>(xl + t * 2 * rs + o);
      }
      y[h][0][i] = *reinterpret_cast<const half8 *>(yh + o);
      y[h][1][i] = *reinterpret_cast<const half8 *>(yl + o);
    }
  };
  f32x16 acc[2] = {};
  if (s0 + wave < s1) {
    fetch(s0 + wave, 0);
    fetch(s0 + wave, 1);
  }
  for (int s = s0 + wave; s < s1; s += 4) {
    f32x16 sum[2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          sum[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[h][t][1][i], y[h][0][i], sum[t], 0, 0, 0);
          sum[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[h][t][0][i], y[h][1][i], sum[t], 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) sum[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[h][t][0][i], y[h][0][i], sum[t], 0, 0, 0);
      if (s + 4 < s1) fetch(s + 4, h);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[t] += sum[t];
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) part[wave][t * 16 + i][lane] = acc[t][i];
  __syncthreads();
}
// A wave finishes half of a 32 x 32 tile: accumulator element f is row 8 (f / 4) + 4 (lane / 32) + f % 4.
// C = fl * sums + fe * E + fd * I of a symmetric result
__device__ __forceinline__ void finish_half(const WaveSums &part, int ti, int tj, const Planes &C, float fl, bool has_e, const Planes &E, float fe, float fd, int n) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, np = C.np;
  const int t = wave >> 1, fi = 2 * ti + t, c = tj * 32 + (lane & 31);
  if (fi > tj) return;
  auto total = [&](int f, int l) { return (part[0][t * 16 + f][l] + part[1][t * 16 + f][l]) + (part[2][t * 16 + f][l] + part[3][t * 16 + f][l]); };
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int f0 = 8 * (wave & 1) + 4 * p, r = fi * 32 + 2 * f0 + 4 * (lane >> 5);
    half4 eh = {}, el = {};
    if (has_e) {                                       // (E is symmetric: its mirror image is one vector)
      const int o = place(np, c, r);
      eh = *reinterpret_cast<const half4 *>(E.hi + o);
      el = *reinterpret_cast<const half4 *>(E.lo() + o);
    }
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float sum = total(f0 + i, lane);
      if (fi == tj && r + i > c) {                     // below the diagonal: what is above it
        const int cc = lane & 31;
        sum = total((cc & 3) + 4 * (cc >> 3), (r + i & 31) + 32 * (cc >> 2 & 1));
      }
      v[i] = fmaf(fl, sum, fmaf(fe, (float)eh[i] + (float)el[i], r + i == c && c < n ? fd : 0.f));
    }
    store_planes4(C, r, c, fi == tj, v);
  }
}

__global__ __launch_bounds__(256, 2) void orth_chain_kernel(ChainArgs a) {
  __shared__ WaveSums part;
  const int id = agx::xcd_logical_id(blockIdx.x, gridDim.x);
  int q = 0;
  while (q + 1 < a.n && id >= a.job[q + 1].first) ++q;
  const ChainJob &j = a.job[q];
  int ti, tj;
  half_tile(id - j.first, j.nt, ti, tj);
  const int64_t np = j.C.np, x = ti * 64 * np, y = tj * 32 * np;
  wave_products(j.L.hi + x, j.L.lo() + x, j.R.hi + y, j.R.lo() + y, 16 * np, 0, (int)(np / BK), part);
  finish_half(part, ti, tj, j.C, __builtin_ldexpf(j.alpha, j.C.e - j.L.e - j.R.e), j.beta != 0.f, j.E,
              __builtin_ldexpf(j.beta, j.C.e - j.E.e), __builtin_ldexpf(j.gamma, j.C.e), j.n);
}

// Gram matrix of the iterate between two phases by the same means: partial tiles as orth_gram_kernel gives them, or (ONE
// slice each) A itself.  18161 x 256 11 us (through LDS, from fp32 lines that every tile splits anew: 15), 256 x 256 5.2 (9),
// 1000 x 4297 38 (44 and 14 for the sum of its slices): a wave lives 20 us and waits for 30% of it, the matrix cores work 6.
struct LinesGramJob {
  Lines x;
  Planes A;
  float *part;
  int32_t nt, slices, per, first;                      // per: steps of 64 lines a slice
};
struct LinesGramArgs {
  LinesGramJob job[AGX_MAX_ORTH];
  int n;
};
template <bool ONE>
__global__ __launch_bounds__(256, 2) void orth_gram_lines_kernel(LinesGramArgs a) {
  __shared__ WaveSums part;
  const int id = agx::xcd_logical_id(blockIdx.x, gridDim.x);
  int q = 0;
  while (q + 1 < a.n && id >= a.job[q + 1].first) ++q;
  const LinesGramJob &j = a.job[q];
  const int tiles = j.nt * (j.nt + 1), slice = ONE ? 0 : (id - j.first) / tiles;
  int ti, tj;
  half_tile((id - j.first) % tiles, j.nt, ti, tj);
  const int64_t rs = 16 * j.x.kp, x = 4 * ti * rs, y = 2 * tj * rs;
  const int s0 = slice * j.per, s1 = min(s0 + j.per, (int)(j.x.kp / BK));
  wave_products(j.x.hi + x, j.x.lo() + x, j.x.hi + y, j.x.lo() + y, rs, s0, s1, part);
  if constexpr (ONE) {
    finish_half(part, ti, tj, j.A, __builtin_ldexpf(1.f, j.A.e - 2 * j.x.e), false, j.A, 0.f, 0.f, 0);
  } else {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = ti * j.nt - ti * (ti - 1) / 2 + tj / 2 - ti;
    float *p = j.part + ((int64_t)tile * j.slices + slice) * T * T + (tj & 1) * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int f = wave * 8 + i, e = f & 15;
      p[((f >> 4) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * T] = (part[0][f][lane] + part[1][f][lane]) + (part[2][f][lane] + part[3][f][lane]);
    }
  }
}

// np <= STEP_NP: rows of a polynomial of A need A alone - r A, (r A) A, ... - so that a workgroup takes 16 rows through
// many products by itself, with A in its waves' registers (256 KB of them at np = 256, 32 columns a wave) and the running
// rows in LDS.  More flops than the symmetric products of whole matrices (6 n^3 a step against 1.5 to 2), but few launches.
//   np = 256, a launch a step: S = a r + b r A + c r A^2, next A = a S + b S A + c S A^2 (four products, r rows of A) and
//     Q = a r + b r A + c r A^2 (two, r rows of the Q before; the first step's Q is S without its A)
//   np <= 128, a launch a phase of up to two steps: u = rows of P_0, then u P_1 with u A_1 = ((u A) P_0) P_0 (twelve products).
//     (Errors of the first of those are multiplied by the later ones: the split's lo.lo products are taken too.  Three
//     products: 23 x 61 off by 1.8e-6, four 1.0e-6, the plain fp32 iteration 0.8e-6.)
// Measured: 8.1 us a step of np = 256 (three launches of whole products: 20), a phase of np = 128 8.1 us and of 64 5.3 us (by
// one workgroup a matrix: 14 and 9).  Bound by the chain of dependent products: 0.4 to 0.8 us each behind 2.4 us of launch and
// 1.5 us until A is in registers.
constexpr int STEP_NP = 256, ROWS = 16;
static_assert(ROWS_PHASE == 128, "the three sides that orth_rows_kernel is made for");
enum { E_U, E_UA, E_UAA, E_W, E_WA, E_Y, E_YA, E_YAA, E_W2, E_WA2, E_COUNT };   // scales of the rows in a phase's panel
struct RowsJob {
  Planes A, An, Q, Qn;
  int32_t n, first;
};
struct RowsArgs {
  RowsJob job[AGX_MAX_ORTH];
  int n;
  int32_t more, has_q;          // a further step follows (A is wanted); Q exists (otherwise the step's own polynomial is Q)
  float a, b, c;
  int32_t e1, eS, e3, q1;       // scale exponents of the running rows: r A, S, S A; of Q's r A
  int32_t steps;                // of a phase
  float a2, b2, c2;             // its second step
  int32_t e[E_COUNT];
};

template <int NP> struct RowsOf {
  static constexpr int LD = NP + 8, CT = NP == 256 ? 2 : 1, KB = NP / 32, BUF = 2 * ROWS * LD;   // (16 rows start in 16 bank groups)
  static constexpr bool FOUR = NP <= ROWS_PHASE;
  typedef f32x4 Result[CT];     // a lane's results: rows 4 g .. of columns col(t)
  half8 bh[CT][KB], bl[CT][KB];
  _Float16 *panel;              // two of [plane][row][LD]
  int buf, ea, i0, pr, pc;      // pr, pc: the row and the first of the eight k's of this thread's piece of a row block
  bool works, piece;            // the wave has columns (np = 64: four of eight do); the thread has a piece
  __device__ __forceinline__ int col(int t) const { return (threadIdx.x >> 6) * 16 * CT + t * 16 + (threadIdx.x & 15); }
  __device__ __forceinline__ int row(int i) const { return 4 * (threadIdx.x >> 4 & 3) + i; }
  __device__ __forceinline__ int mine() const { return i0 * NP + threadIdx.x * 8; }
  // the rows from R, and all of A
  __device__ __forceinline__ RowsOf(const Planes &R, const Planes &A, int first_row, _Float16 *lds) : panel(lds), buf(0), ea(A.e), i0(first_row) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    works = wave * 16 * CT < NP;
    piece = (int)threadIdx.x < 2 * NP;
    placed(NP, threadIdx.x, pr, pc);
    half8 rh, rl;
    if (piece) {
      rh = *reinterpret_cast<const half8 *>(R.hi + mine());
      rl = *reinterpret_cast<const half8 *>(R.lo() + mine());
    }
    // (k runs in an order of its own, the same for both operands: a wave's vectors are what place() keeps together)
    if (works)
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          const int o = (wave * CT + t) * 16 * NP + k * 512 + lane * 8;
          bh[t][k] = *reinterpret_cast<const half8 *>(A.hi + o);
          bl[t][k] = *reinterpret_cast<const half8 *>(A.lo() + o);
        }
    if (piece) {
      *reinterpret_cast<half8 *>(&panel[pr * LD + pc]) = rh;
      *reinterpret_cast<half8 *>(&panel[ROWS * LD + pr * LD + pc]) = rl;
    }
    __syncthreads();
  }
  __device__ __forceinline__ _Float16 *plane(int lo) const { return panel + buf * BUF + lo * ROWS * LD; }
  __device__ __forceinline__ void values(int e, Result &out) const {    // the rows in the panel, of scale e
    if (!works) return;
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int o = row(i) * LD + col(t);
        out[t][i] = __builtin_ldexpf((float)plane(0)[o] + (float)plane(1)[o], -e);
      }
  }
  __device__ __forceinline__ void multiply(int e, Result &out) const {  // out = (rows in the panel, of scale e) . A
    if (!works) return;
    const int at = (threadIdx.x & 15) * LD + (threadIdx.x >> 4 & 3) * 16;
    const _Float16 *ph = plane(0) + at, *pl = plane(1) + at;
    f32x4 acc[CT] = {};
#pragma unroll
    for (int k = 0; k < KB; k += KB < 4 ? KB : 4) {
      f32x4 sum[CT] = {};
      half8 x[4];
#pragma unroll
      for (int h = 0; h < (KB < 4 ? KB : 4); ++h) {
        const int o = (k + h >> 1) * 64 + (h & 1) * 8;
        x[h] = *reinterpret_cast<const half8 *>(ph + o);
        const half8 y = *reinterpret_cast<const half8 *>(pl + o);
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          if (FOUR) sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, bl[t][k + h], sum[t], 0, 0, 0);
          sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, bh[t][k + h], sum[t], 0, 0, 0);
          sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[h], bl[t][k + h], sum[t], 0, 0, 0);
        }
      }
#pragma unroll
      for (int h = 0; h < (KB < 4 ? KB : 4); ++h)
#pragma unroll
        for (int t = 0; t < CT; ++t) sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[h], bh[t][k + h], sum[t], 0, 0, 0);
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t] += sum[t];
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) out[t] = scale4(acc[t], -e - ea);
  }
  __device__ __forceinline__ void put(const Result &r, int e) {         // rows into the other panel, which is then the current one
    buf ^= 1;
    if (works)
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        half4 h, l;
        split4(scale4(r[t], e), h, l);
        store_pairs4(plane(0), LD, row(0), col(t), h);
        store_pairs4(plane(1), LD, row(0), col(t), l);
      }
    __syncthreads();
  }
  __device__ __forceinline__ void write(const Planes &m) const {        // the current panel
    if (!piece) return;
    *reinterpret_cast<half8 *>(m.hi + mine()) = *reinterpret_cast<const half8 *>(plane(0) + pr * LD + pc);
    *reinterpret_cast<half8 *>(m.lo() + mine()) = *reinterpret_cast<const half8 *>(plane(1) + pr * LD + pc);
  }
  // out = a v + b v1 + c v2, a on the diagonal where v is the identity's rows
  template <class V>
  __device__ __forceinline__ void combine(float a, V v, float b, const Result &v1, float c, const Result &v2, Result &out) const {
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) out[t][i] = fmaf(a, v(t, i), fmaf(b, v1[t][i], c * v2[t][i]));
  }
  __device__ __forceinline__ void combine(float a, const Result &v, float b, const Result &v1, float c, const Result &v2, Result &out) const {
    combine(a, [&](int t, int i) { return v[t][i]; }, b, v1, c, v2, out);
  }
  // rows of P_0: a I + b r + c r A, r = rows of A in the panel
  __device__ __forceinline__ void polynomial(const RowsArgs &p, int n, const Result &r, const Result &x1, Result &out) const {
    combine(p.a, [&](int t, int i) { return i0 + row(i) == col(t) && col(t) < n ? 1.f : 0.f; }, p.b, r, p.c, x1, out);
  }
};

// one step of np = 256; local: 16 workgroups for rows of A (where they or the first Q are wanted), then 16 for rows of Q
__device__ __forceinline__ void rows_step(const RowsArgs &a, const RowsJob &j, int local, _Float16 *lds) {
  typedef RowsOf<STEP_NP> R;
  const bool rows_of_q = local >= STEP_NP / ROWS;
  if (rows_of_q ? !a.has_q : a.has_q && !a.more) return;
  const Planes &from = rows_of_q ? j.Q : j.A;
  R x(from, j.A, local % (STEP_NP / ROWS) * ROWS, lds);
  R::Result r, x1, x2, s;
  x.values(from.e, r);
  x.multiply(from.e, x1);
  if (!rows_of_q && !a.has_q) {
    x.polynomial(a, j.n, r, x1, s);
    x.put(s, j.Qn.e);
    x.write(j.Qn);
    if (!a.more) return;
  }
  const int e1 = rows_of_q ? a.q1 : a.e1;
  x.put(x1, e1);
  x.multiply(e1, x2);
  x.combine(a.a, r, a.b, x1, a.c, x2, s);
  if (rows_of_q) {
    x.put(s, j.Qn.e);
    x.write(j.Qn);
    return;
  }
  x.put(s, a.eS);
  x.multiply(a.eS, x1);
  x.put(x1, a.e3);
  x.multiply(a.e3, x2);
  x.combine(a.a, s, a.b, x1, a.c, x2, s);
  x.put(s, j.An.e);
  // the rows from the diagonal on, and their mirror image behind it
  const int from_diagonal = x.pc - x.i0;
  if (from_diagonal >= ROWS) {
    x.write(j.An);
  } else if (from_diagonal >= 0) {                     // (the square on the diagonal: symmetric from what is above it)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = from_diagonal + k, o = min(x.pr, c) * R::LD + x.i0 + max(x.pr, c);
      j.An.hi[x.mine() + k] = x.plane(0)[o];
      j.An.lo()[x.mine() + k] = x.plane(1)[o];
    }
  }
#pragma unroll
  for (int t = 0; t < R::CT; ++t) {
    if (x.col(t) >= x.i0 + ROWS) {
      half4 h, l;
      split4(scale4(s[t], j.An.e), h, l);
      const int o = place(STEP_NP, x.col(t), x.i0 + x.row(0));
      *reinterpret_cast<half4 *>(j.An.hi + o) = h;
      *reinterpret_cast<half4 *>(j.An.lo() + o) = l;
    }
  }
}
// a phase of np <= 128, one workgroup for 16 rows of its Q
template <int NP>
__device__ __forceinline__ void rows_phase(const RowsArgs &a, const RowsJob &j, int local, _Float16 *lds) {
  typedef RowsOf<NP> R;
  R x(j.A, j.A, local * ROWS, lds);
  typename R::Result u, v, v1, v2, y1;
  x.values(j.A.e, v);
  x.multiply(j.A.e, v1);
  x.polynomial(a, j.n, v, v1, u);
  if (a.steps > 1) {
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {                      // u A_1, (u A_1) A_1
      const int32_t *e = a.e + 5 * k;
      if (k == 0) x.put(u, e[0]);
      else x.put(y1, e[0]);
      x.multiply(e[0], v);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {                    // . P_0, twice
        x.put(v, e[1 + 2 * i]);
        x.multiply(e[1 + 2 * i], v1);
        x.put(v1, e[2 + 2 * i]);
        x.multiply(e[2 + 2 * i], v2);
        x.combine(a.a, v, a.b, v1, a.c, v2, v);
      }
      if (k == 0)
#pragma unroll
        for (int t = 0; t < R::CT; ++t) y1[t] = v[t];
    }
    x.combine(a.a2, u, a.b2, y1, a.c2, v, u);
  }
  x.put(u, j.Qn.e);
  x.write(j.Qn);
}
__global__ __launch_bounds__(512, 2) void orth_rows_kernel(RowsArgs a) {
  __shared__ __align__(16) _Float16 lds[2 * RowsOf<STEP_NP>::BUF];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const RowsJob &j = a.job[q];
  const int local = (int)blockIdx.x - j.first;
  if (j.A.np == STEP_NP) rows_step(a, j, local, lds);
  else if (j.A.np == ROWS_PHASE) rows_phase<ROWS_PHASE>(a, j, local, lds);
  else rows_phase<T>(a, j, local, lds);
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
  int32_t rows, cols, tall, dtype, otype, e, nb, muon, lines, first;   // lines: of X, up to where they are wanted
  Lines from, to;               // the iterate instead of x / out where they are there
};
static_assert(sizeof(ApplyJob) * AGX_MAX_ORTH <= 4000, "kernel argument size");
struct ApplyArgs {
  ApplyJob job[AGX_MAX_ORTH];
  int n, per;                   // per: groups of lines a workgroup (orth_panel_kernel)
};

// from the scaled product to Y (in 64 bits where the factor leaves fp32's normal range: tiny matrices)
struct Factor {
  double f;
  float ff;
  bool plain;
  __device__ __forceinline__ Factor(const ApplyJob &j, int e) : f(ldexp(j.invd ? *j.invd : ldexp(1.0, -e), (j.to.hi ? j.to.e : 0) - j.Q.e)), ff((float)f) {
    plain = __builtin_amdgcn_readfirstlane((fabsf(ff) >= 1.2e-38f && fabsf(ff) <= 1e38f) || f == 0.0);
  }
};
// a wave's 32 x 32 results of it, from row r0 and column c0 of Y on (scalar row pointers, one offset a lane)
template <typename O, bool MUON, bool INSIDE>
__device__ __forceinline__ void write_tile(O *o, const ApplyJob &j, const f32x16 &acc, int r0, int c0) {
  const int lane = threadIdx.x & 63, lr = 4 * (lane >> 5), left = j.rows - r0 - lr, ldo = (int)j.ldo, off = lr * ldo + (lane & 31);
  const bool column = (lane & 31) < j.cols - c0;
  const float decay = j.decay, step = j.step;
  o += (int64_t)r0 * j.ldo + c0;
  auto row = [](int k) { return 8 * (k >> 2) + (k & 3); };
  auto ok = [&](int k) { return INSIDE || (row(k) < left && column); };
  f32x16 y = acc;
  if constexpr (MUON) {
#pragma unroll
    for (int k = 0; k < 16; ++k) y[k] = ok(k) ? (o + row(k) * ldo)[off] : 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) y[k] = decay * y[k] - step * acc[k];
  }
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (ok(k)) (o + row(k) * ldo)[off] = (O)y[k];
}
template <bool INSIDE>
__device__ __forceinline__ void write_tile(const ApplyJob &j, const f32x16 &acc, int r0, int c0) {
  if (j.muon) write_tile<float, true, INSIDE>(reinterpret_cast<float *>(j.out), j, acc, r0, c0);
  else if (j.otype == AGX_F32) write_tile<float, false, INSIDE>(reinterpret_cast<float *>(j.out), j, acc, r0, c0);
  else write_tile<__bf16, false, INSIDE>(reinterpret_cast<__bf16 *>(j.out), j, acc, r0, c0);
}
__device__ __forceinline__ void multiply(f32x16 &acc, const Factor &f) {
  if (f.plain) {
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] *= f.ff;
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = (float)((double)acc[k] * f.f);
  }
}
// the same of lines l0.. and values c0.. into the iterate: four lines of a value are neighbours
__device__ __forceinline__ void finish_lines(const ApplyJob &j, const Factor &f, f32x16 acc, int l0, int c0) {
  const int lane = threadIdx.x & 63;
  multiply(acc, f);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    half4 h, l;
    split4(f32x4{acc[4 * p], acc[4 * p + 1], acc[4 * p + 2], acc[4 * p + 3]}, h, l);
    const int64_t o = j.to.at(c0 + (lane & 31), l0 + 8 * p + 4 * (lane >> 5));
    *reinterpret_cast<half4 *>(j.to.hi + o) = h;
    *reinterpret_cast<half4 *>(j.to.lo() + o) = l;
  }
}
__device__ __forceinline__ void finish_tile(const ApplyJob &j, const Factor &f, f32x16 acc, int r0, int c0) {
  multiply(acc, f);
  // (tiles inside the matrix, nearly all, without a condition per element: each would wait for what is in flight)
  if (r0 + 32 <= j.rows && c0 + 32 <= j.cols) write_tile<true>(j, acc, r0, c0);
  else write_tile<false>(j, acc, r0, c0);
}

// lines tl * 64.. by values tn * 64..: XQ with the lines as the result's rows, as a tall matrix and the iterate want it
template <bool XQ, class L>
__device__ __forceinline__ f32x16 apply_tile(const ApplyJob &j, L &lx, int tl, int tn, int &e, uint32_t *red, _Float16 *lds) {
  LoadPlanes lq(j.Q);
  auto late = [&] { lx.e = e = j.nb ? scale_exponent(j.maxb, j.nb, red) : j.e; };
  if constexpr (XQ) return tile_product(lx, lq, (int64_t)tl * T, (int64_t)tn * T, 0, j.Q.np, lds, false, late);
  else return tile_product(lq, lx, (int64_t)tn * T, (int64_t)tl * T, 0, j.Q.np, lds, false, late);
}
template <class L>
__device__ __forceinline__ void apply_job(const ApplyJob &j, L lx, int tl, int tn, uint32_t *red, _Float16 *lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), a = (wave >> 1) * 32, b = (wave & 1) * 32;
  int e;
  if (j.tall || j.to.hi) {
    const f32x16 acc = apply_tile<true>(j, lx, tl, tn, e, red, lds);
    if (j.to.hi) finish_lines(j, Factor(j, e), acc, tl * T + a, tn * T + b);
    else finish_tile(j, Factor(j, e), acc, tl * T + a, tn * T + b);
  } else {
    const f32x16 acc = apply_tile<false>(j, lx, tl, tn, e, red, lds);
    finish_tile(j, Factor(j, e), acc, tn * T + a, tl * T + b);
  }
}

template <int KIND>
__global__ __launch_bounds__(256, 4) void orth_apply_kernel(ApplyArgs a) {
  __shared__ __align__(16) _Float16 lds[4 * PL];
  __shared__ uint32_t red[4];
  // (tiles that read the same part of X follow each other on one XCD)
  const int id = agx::xcd_logical_id(blockIdx.x, gridDim.x);
  int q = 0;
  while (q + 1 < a.n && id >= a.job[q + 1].first) ++q;
  const ApplyJob &j = a.job[q];
  const int tns = j.to.hi ? j.Q.np / T : ((j.tall ? j.cols : j.rows) + T - 1) / T, tl = (id - j.first) / tns, tn = (id - j.first) % tns;
  if constexpr (KIND == ITERATE) {
    LoadLines lx;
    lx.x = &j.from;
    apply_job(j, lx, tl, tn, red, lds);
  } else {
    auto is = [&](int kind) { return KIND == ANY ? is_kind(kind, j.tall, j.dtype) : KIND == kind; };
    auto user = [&](auto lx) {
      lx.p = reinterpret_cast<decltype(lx.p)>(j.x);
      lx.ld = j.ldx; lx.rows = j.tall ? j.rows : j.cols; lx.kmax = j.tall ? j.cols : j.rows;
      apply_job(j, lx, tl, tn, red, lds);
    };
    if (is(0)) user(LoadK<float>{});
    else if (is(1)) user(LoadT<float>{});
    else if (is(2)) user(LoadK<__bf16>{});
    else user(LoadT<__bf16>{});
  }
}

// The same for np <= PANEL_NP.  Its eight waves hold all of Q in registers (32 columns each, over all of k; at np = 128 and 64
// two and four groups of waves hold it), and the lines of X - rows of a tall matrix, columns of a wide one - go by in groups
// of 8192 / np through two LDS buffers, converted once, the next group's loads in flight: one workgroup a CU.  18161 x 256
// 17.3 us (tiles of 64 x 64 as above: 23 us; its 37 MB take 7.4 us at 5 TB/s), 3 groups a workgroup of 2.7 us each: 1.3 us
// of matrix products, then the results' way out and the next group's way in, which a barrier a group keeps apart.
constexpr int PANEL_NP = 256, PANEL_LDS = 2 * 2 * 128 * (64 + 8) * 2;    // (np = 64 has the most padding)
// a group's loads and LDS writes: 16 elements a thread, raw until they are stored
template <typename E, bool TALL, int NP> struct PanelLines {
  static constexpr int GL = 8192 / NP, LD = NP + 8;    // (rows that start in 16 different bank groups)
  static constexpr bool two = sizeof(E) == 4;
  using V = typename Vec4<E>::type;
  V v[4];
  // tall: four vectors along k; wide: four k's of four lines
  static __device__ __forceinline__ int line(int q) { return TALL ? (threadIdx.x + 512 * q) / (NP / 4) : threadIdx.x % (GL / 4) * 4; }
  static __device__ __forceinline__ int k(int q) { return TALL ? threadIdx.x % (NP / 4) * 4 : threadIdx.x / (GL / 4) * 4 + q; }
  __device__ __forceinline__ void fetch(const ApplyJob &j, int l0) {
    const int lines = TALL ? j.rows : j.cols, n = TALL ? j.cols : j.rows, ld = (int)j.ldx;
    const E *b = reinterpret_cast<const E *>(j.x) + (TALL ? (int64_t)l0 * j.ldx : (int64_t)l0);
    if (l0 + GL <= lines && n == NP) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const V *>(b + (TALL ? line(q) * ld + k(q) : k(q) * ld + line(q)));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int l = line(q) + (TALL ? 0 : i), kk = k(q) + (TALL ? i : 0);
          v[q][i] = l0 + l < lines && kk < n ? b[TALL ? l * ld + kk : kk * ld + l] : (E)0.f;
        }
    }
  }
  __device__ __forceinline__ void store(_Float16 *hi, _Float16 *lo, int e) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      half4 h, l;
      if (TALL) split4(scale4(f32x4{(float)v[q][0], (float)v[q][1], (float)v[q][2], (float)v[q][3]}, e), h, l);
      else split4(scale4(f32x4{(float)v[0][q], (float)v[1][q], (float)v[2][q], (float)v[3][q]}, e), h, l);
      const int o = TALL ? line(q) * LD + k(q) : (line(0) + q) * LD + k(0);
      *reinterpret_cast<half4 *>(hi + o) = h;
      if (sizeof(E) == 4) *reinterpret_cast<half4 *>(lo + o) = l;
    }
  }
};
// the same from the iterate: blocks of four values of four lines
template <int NP> struct PanelIterate {
  static constexpr int GL = 8192 / NP, LD = NP + 8;
  static constexpr bool two = true;
  half4 vh[4], vl[4];                                  // [value][line]
  static __device__ __forceinline__ int line() { return threadIdx.x % (GL / 4) * 4; }
  static __device__ __forceinline__ int k() { return threadIdx.x / (GL / 4) * 4; }
  __device__ __forceinline__ void fetch(const ApplyJob &j, int l0) {
    const int l = l0 + line();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      vh[q] = vl[q] = half4{};
      if (l < j.from.kp) {
        const int64_t o = j.from.at(k() + q, l);
        vh[q] = *reinterpret_cast<const half4 *>(j.from.hi + o);
        vl[q] = *reinterpret_cast<const half4 *>(j.from.lo() + o);
      }
    }
  }
  __device__ __forceinline__ void store(_Float16 *hi, _Float16 *lo, int) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int o = (line() + q) * LD + k();
      *reinterpret_cast<half4 *>(hi + o) = half4{vh[0][q], vh[1][q], vh[2][q], vh[3][q]};
      *reinterpret_cast<half4 *>(lo + o) = half4{vl[0][q], vl[1][q], vl[2][q], vl[3][q]};
    }
  }
};
// XQ: as in apply_tile
template <class X, int NP, bool XQ>
__device__ __forceinline__ void panel_groups(const ApplyJob &j, int per, uint32_t *red, _Float16 *lds) {
  constexpr int CG = NP / 32, NB = NP / 32, PLANE = X::GL * X::LD;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cg = wave % CG, rg = wave / CG;
  const int g0 = ((int)blockIdx.x - j.first) * per, g1 = min(g0 + per, (j.lines + X::GL - 1) / X::GL);
  X x;
  x.fetch(j, g0 * X::GL);
  // (k runs in an order of its own, the same for both operands: a lane's two vectors of a block are neighbours in memory)
  half8 qh[NB][2], ql[NB][2];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int o = place(NP, cg * 32 + (lane & 31), b * 32 + (lane >> 5) * 16 + i * 8);
      qh[b][i] = *reinterpret_cast<const half8 *>(j.Q.hi + o);
      ql[b][i] = *reinterpret_cast<const half8 *>(j.Q.lo() + o);
    }
  const int e = j.nb ? scale_exponent(j.maxb, j.nb, red) : j.e;
  x.store(lds, lds + PLANE, e);
  const Factor f(j, e);
  for (int g = g0, buf = 0; g < g1; ++g, buf ^= 1) {   // (one barrier a group: a buffer is written a group after it was read)
    if (g + 1 < g1) x.fetch(j, (g + 1) * X::GL);
    __syncthreads();
    const _Float16 *xl = lds + buf * 2 * PLANE + (rg * 32 + (lane & 31)) * X::LD + (lane >> 5) * 16;
    auto at = [&](int o) { return *reinterpret_cast<const half8 *>(xl + o); };
    f32x16 acc = {};
#pragma unroll
    for (int s = 0; s < NB; s += 2) {                  // (steps of 64 k, as in tile_product)
      f32x16 sum = {};
      auto mul = [&](half8 xv, half8 qv) {
        sum = XQ ? __builtin_amdgcn_mfma_f32_32x32x16_f16(xv, qv, sum, 0, 0, 0)
                 : __builtin_amdgcn_mfma_f32_32x32x16_f16(qv, xv, sum, 0, 0, 0);
      };
#pragma unroll
      for (int b = s; b < s + 2; ++b) {
        const half8 x0 = at(b * 32), x1 = at(b * 32 + 8);
        mul(x0, ql[b][0]);
        mul(x1, ql[b][1]);
        if (X::two) {
          mul(at(PLANE + b * 32), qh[b][0]);
          mul(at(PLANE + b * 32 + 8), qh[b][1]);
        }
        mul(x0, qh[b][0]);
        mul(x1, qh[b][1]);
      }
      acc += sum;
      asm volatile("" : "+v"(acc));                    // (put off to the epilogue, the sums would not fit the registers)
    }
    const int l = g * X::GL + rg * 32, c = cg * 32;
    if (l < j.lines) {
      if (XQ && j.to.hi) finish_lines(j, f, acc, l, c);
      else if (c < (XQ ? j.cols : j.rows)) finish_tile(j, f, acc, XQ ? l : c, XQ ? c : l);
    }
    if (g + 1 < g1) x.store(lds + (buf ^ 1) * 2 * PLANE, lds + (buf ^ 1) * 2 * PLANE + PLANE, e);
  }
}
template <class F, int NP>
__device__ __forceinline__ void panel_order(const ApplyJob &j, int per, uint32_t *red, _Float16 *lds) {
  if (F::tall || j.tall || j.to.hi) panel_groups<typename F::template X<NP>, NP, true>(j, per, red, lds);
  else if constexpr (!F::tall) panel_groups<typename F::template X<NP>, NP, false>(j, per, red, lds);
}
template <class F>
__device__ __forceinline__ void panel_job(const ApplyJob &j, int per, uint32_t *red, _Float16 *lds) {
  if (j.Q.np == 64) panel_order<F, 64>(j, per, red, lds);
  else if (j.Q.np == 128) panel_order<F, 128>(j, per, red, lds);
  else panel_order<F, 256>(j, per, red, lds);
}
template <typename E, bool TALL> struct FromUser {
  static constexpr bool tall = TALL;
  template <int NP> using X = PanelLines<E, TALL, NP>;
};
struct FromIterate {
  static constexpr bool tall = false;                  // (either, see panel_order)
  template <int NP> using X = PanelIterate<NP>;
};
template <int KIND>
__global__ __launch_bounds__(512, 2) void orth_panel_kernel(ApplyArgs a) {
  extern __shared__ _Float16 lds[];
  __shared__ uint32_t red[8];
  int q = 0;
  while (q + 1 < a.n && (int)blockIdx.x >= a.job[q + 1].first) ++q;
  const ApplyJob j = a.job[q];                         // (by value: a reference into the arguments would go through scratch)
  if constexpr (KIND == ITERATE) {
    panel_job<FromIterate>(j, a.per, red, lds);
  } else {
    auto is = [&](int kind) { return KIND == ANY ? is_kind(kind, j.tall, j.dtype) : KIND == kind; };
    if (is(0)) panel_job<FromUser<float, true>>(j, a.per, red, lds);
    else if (is(1)) panel_job<FromUser<float, false>>(j, a.per, red, lds);
    else if (is(2)) panel_job<FromUser<__bf16, true>>(j, a.per, red, lds);
    else panel_job<FromUser<__bf16, false>>(j, a.per, red, lds);
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
  bool square_wide = false;   // a square matrix is taken as the call's others are
  bool tall() const { return rows > cols || (rows == cols && !square_wide); }
  int n() const { return std::min(rows, cols); }
  int64_t K() const { return std::max(rows, cols); }
  int64_t kp() const { return (K() + BK - 1) / BK * BK; }
  int np() const { return n() <= T ? T : n() <= 2 * T ? 2 * T : n() <= STEP_NP ? STEP_NP : agx::cdiv(n(), T) * T; }
  int nt() const { return agx::cdiv(n(), T); }                   // tiles along the small side that hold anything
  int tiles() const { return nt() * (nt() + 1) / 2; }
};

struct Layout {       // workspace of one job, in bytes from its start
  int64_t maxb, squares, invd, mat[5], part, x[2], u, end;
  int slices;
  int64_t kper;
};
int64_t up256(int64_t v) { return (v + 255) & ~(int64_t)255; }

// what all matrices of a launch are (orth_gram_kernel), one more of them taken in
int joined_kind(int kind, bool tall, int dtype) {
  const int k = (tall ? 0 : 1) + (dtype != AGX_F32 ? 2 : 0);
  return kind < 0 || kind == k ? k : ANY;
}
// calls f with the kind as a constant: what a caller's matrices are, or the iterate's planes too
template <class F> void by_user_kind(int kind, F f) {
  switch (kind) {
    case 0: f(std::integral_constant<int, 0>{}); break;
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    default: f(std::integral_constant<int, ANY>{});
  }
}
template <class F> void by_kind(int kind, F f) {
  if (kind == ITERATE) f(std::integral_constant<int, ITERATE>{});
  else by_user_kind(kind, f);
}

int64_t longest(const Job *jobs, int n) {               // steps of the longest of a call's Gram products
  int64_t k = 0;
  for (int i = 0; i < n; ++i) k = std::max(k, agx::cdiv64(jobs[i].K(), BK));
  return k;
}
// slices of a Gram product.  Up to ONE_SLICE steps one, whose launch gives the matrix itself (256 x 256 92 us instead of 96,
// 100 x 60 57 instead of 64; 7 steps in one slice: 400 x 400 173 us instead of 156).  Beyond: two workgroups a CU for tall
// matrices and four for wide ones, over all of the call's matrices - each writes, and the next launch reads, a whole tile
// (18161 x 256: 2, 3, 4 a CU 152, 157, 157 us; 1000 x 4297 419, 397, 387; GTEx generator's Muon step 188, 182, 177).
// most_steps: longest().
void plan(const Job &j, int total_tiles, int64_t most_steps, int phases, bool need_u, Layout &l) {
  const int tiles = j.tiles();
  const int64_t ksteps = agx::cdiv64(j.K(), BK);
  const int64_t want = std::max<int64_t>(1, (int64_t)agx::num_cus() * (j.rows >= j.cols ? TALL_BLOCKS : WIDE_BLOCKS) / std::max(1, total_tiles));
  l.kper = std::max<int64_t>(std::min<int64_t>(ksteps, most_steps <= ONE_SLICE ? ONE_SLICE : 2), agx::cdiv64(ksteps, want)) * BK;
  l.slices = (int)agx::cdiv64(j.K(), l.kper);
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = up256(off + bytes); return o; };
  l.maxb = take(MAXB * 4);
  l.squares = take(MAXB * 8);
  l.invd = take(8);
  for (int64_t &m : l.mat) m = take((int64_t)j.np() * j.np() * 4);
  l.part = take((int64_t)tiles * l.slices * T * T * 4);
  for (int k = 0; k < 2; ++k) l.x[k] = phases > 1 + k ? take(j.np() * j.kp() * 4) : 0;
  l.u = need_u ? take((int64_t)j.rows * j.cols * 4) : 0;
  l.end = off;
}
// Steps between two Gram matrices.  Error against 64 bits over the plain fp32 iteration's (gradients of a few strong directions
// and noise): sides up to 256, of 19 x 201 to 18161 x 256, three steps 2.9 in the mean and up to 7.3, two 1.1 and up to 1.8;
// sides above, whose fp32 sums are longer, three steps 0.6 to 0.8.  Two steps cost 18161 x 256 a fifth of its time, 1000 x 4297
// as much.
int phase_of(const Job *jobs, int n) {
  for (int i = 0; i < n; ++i)
    if (jobs[i].np() <= PANEL_NP) return 2;
  return PHASE;
}

int64_t ws_bytes(const Job *jobs, int n, int steps, bool need_u) {
  int tiles = 0;
  for (int i = 0; i < n; ++i) tiles += jobs[i].tiles();
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    Layout l;
    plan(jobs[i], tiles, longest(jobs, n), agx::cdiv(steps, phase_of(jobs, n)), need_u, l);
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
  for (int i = 0; i < n; ++i) {
    const Job &j = jobs[i];
    const int size = j.dtype == AGX_F32 ? 4 : 2;
    const agx::Region used{ws, 1, need, need, 1};
    for (const agx::Region &r : {agx::Region{j.x, j.rows, j.cols, j.ldx, size}, agx::Region{j.out, j.rows, j.cols, j.ldo, size},
                                 agx::Region{j.m, j.rows, j.cols, j.ldm, size}})
      AGX_CHECK_ARG(!agx::overlap(used, r), "%s: the workspace overlaps matrix %d", who, i);
  }
  int tiles = 0, wide = 0;
  for (int i = 0; i < n; ++i) {
    tiles += jobs[i].tiles();
    wide += (jobs[i].rows < jobs[i].cols) - (jobs[i].rows > jobs[i].cols);
  }
  for (int i = 0; i < n; ++i) jobs[i].square_wide = wide > 0;
  const int phase = phase_of(jobs, n), phases = agx::cdiv(o->steps, phase);
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
      plan(j, tiles, longest(jobs, n), phases, need_u && j.muon, lay[i]);
      base[i] = ws;
      ws += lay[i].end;
      nb[i] = (int)std::min<int64_t>(MAXB, agx::cdiv64((int64_t)j.rows * agx::cdiv(j.cols, 4), 512));
      gx = std::max(gx, nb[i]);
      PrepJob &p = pa.job[i];
      p.x = j.x; p.ldx = j.ldx; p.rows = j.rows; p.cols = j.cols; p.dtype = j.dtype; p.nb = nb[i];
      p.maxb = reinterpret_cast<uint32_t *>(base[i] + lay[i].maxb);
      p.squares = reinterpret_cast<double *>(base[i] + lay[i].squares);
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
  auto planes = [&](int i, int k, int e) {
    Planes p;
    p.hi = reinterpret_cast<_Float16 *>(base[i] + lay[i].mat[k]);
    p.e = e;
    p.np = jobs[i].np();
    return p;
  };
  // matrices of np <= ROWS_PHASE take a launch a phase, of np = STEP_NP a launch a step, the others three a step
  auto by_products = [&](int i) { return jobs[i].np() > STEP_NP; };
  bool any_phases = false, any_steps = false, any_products = false;
  for (int i = 0; i < n; ++i) {
    any_phases = any_phases || jobs[i].np() <= ROWS_PHASE;
    any_steps = any_steps || jobs[i].np() == STEP_NP;
    any_products = any_products || by_products(i);
  }
  double s = 1.0;       // bound on the iterate's singular values (|X_0| <= |X_0|_F <= 1)
  for (int ph = 0, k = 0; ph < phases; ++ph) {
    const bool first = ph == 0, last = ph == phases - 1;
    const int ex = exponent_for(s);                 // scale of the iterate (later phases)
    auto iterate = [&](int phase_number, int i, int e) {             // what that phase leaves
      Lines l;
      l.hi = reinterpret_cast<_Float16 *>(base[i] + lay[i].x[phase_number & 1]);
      l.kp = jobs[i].kp();
      l.e = e;
      l.np = jobs[i].np();
      return l;
    };
    auto add_slices = [&](ReduceArgs &ra, int blocks, int pieces) -> int {
      if (pieces == 8) hipLaunchKernelGGL(orth_reduce_kernel<4>, dim3(blocks), dim3(reduce_threads<4>()), 0, st, ra);
      else hipLaunchKernelGGL(orth_reduce_kernel<32>, dim3(blocks), dim3(reduce_threads<32>()), 0, st, ra);
      AGX_LAUNCH_CHECK();
      return AGX_OK;
    };
    if (first) {
      GramArgs ga;
      ReduceArgs ra;
      ga.n = ra.n = n;
      ga.eps = ra.eps = o->eps;
      int gb = 0, rb = 0, kind = -1, most = 0;
      for (int i = 0; i < n; ++i) most = std::max(most, lay[i].slices);
      const bool one = most == 1;                       // nothing to add
      const int pieces = most > FEW_SLICES ? 8 : 1;     // of a square of 32 x 32
      for (int i = 0; i < n; ++i) {
        const Job &j = jobs[i];
        const Layout &l = lay[i];
        const int nt = one ? j.np() / T : j.nt();
        GramJob &g = ga.job[i];
        g.x = j.x; g.ld = j.ldx; g.K = j.K(); g.kper = l.kper; g.n = j.n(); g.nt = nt; g.slices = l.slices; g.tall = j.tall();
        g.dtype = j.dtype; g.nb = nb[i];
        g.maxb = reinterpret_cast<const uint32_t *>(base[i] + l.maxb);
        g.part = reinterpret_cast<float *>(base[i] + l.part);
        g.squares = reinterpret_cast<const double *>(base[i] + l.squares);
        g.invd = reinterpret_cast<double *>(base[i] + l.invd);
        g.A = planes(i, 0, exponent_for(s * s));
        g.first = gb;
        gb += nt * (nt + 1) / 2 * l.slices;
        kind = joined_kind(kind, g.tall, g.dtype);
        ReduceJob &r = ra.job[i];
        r.part = g.part; r.squares = g.squares; r.maxb = g.maxb; r.invd = g.invd;
        r.A = g.A; r.nt = nt; r.slices = l.slices; r.e = 0; r.nb = nb[i];
        r.normalise = true; r.first = rb;
        rb += j.np() / 32 * (j.np() / 32 + 1) / 2 * pieces;
      }
      by_user_kind(kind, [&](auto k) {
        if (one) hipLaunchKernelGGL((orth_gram_kernel<decltype(k)::value, true>), dim3(gb), dim3(256), 0, st, ga);
        else hipLaunchKernelGGL((orth_gram_kernel<decltype(k)::value, false>), dim3(gb), dim3(256), 0, st, ga);
      });
      AGX_LAUNCH_CHECK();
      if (!one) AGX_TRY(add_slices(ra, rb, pieces));
    } else {
      LinesGramArgs ga;
      ReduceArgs ra;
      memset(&ga, 0, sizeof(ga));
      memset(&ra, 0, sizeof(ra));
      ga.n = ra.n = n;
      int gb = 0, rb = 0, most = 0;
      for (int i = 0; i < n; ++i) {
        const int steps_i = (int)(jobs[i].kp() / BK), want = std::max(1, agx::num_cus() * LINES_BLOCKS / std::max(1, 2 * tiles));
        // (four steps at least, one a wave; no more slices than the first phase had room for.  Two workgroups a CU, as many as
        //  fit it: 18161 x 256 1, 2, 3, 4 of them 146, 147, 150, 152 us, GTEx generator's Muon step 181, 168, 173, 169.  Up to
        //  16 steps in one slice: 1024 x 1024 256 us, with slices 263; up to 32 makes no difference at 640 x 2000.)
        const int per = longest(jobs, n) <= ONE_SLICE_LINES ? steps_i
                                                           : std::max({std::min(steps_i, 4), agx::cdiv(steps_i, want), agx::cdiv(steps_i, lay[i].slices)});
        ga.job[i].per = per;
        ga.job[i].slices = agx::cdiv(steps_i, per);
        most = std::max(most, ga.job[i].slices);
      }
      const bool one = most == 1;
      const int pieces = most > FEW_SLICES ? 8 : 1;
      for (int i = 0; i < n; ++i) {
        const Job &j = jobs[i];
        LinesGramJob &g = ga.job[i];
        g.x = iterate(ph - 1, i, ex);
        g.A = planes(i, 0, exponent_for(s * s));
        g.part = reinterpret_cast<float *>(base[i] + lay[i].part);
        g.nt = one ? j.np() / T : j.nt();
        g.first = gb;
        gb += g.nt * (g.nt + 1) * g.slices;
        ReduceJob &r = ra.job[i];
        r.part = g.part; r.A = g.A; r.nt = g.nt; r.slices = g.slices; r.e = ex; r.first = rb;
        rb += j.np() / 32 * (j.np() / 32 + 1) / 2 * pieces;
      }
      if (one) hipLaunchKernelGGL(orth_gram_lines_kernel<true>, dim3(gb), dim3(256), 0, st, ga);
      else hipLaunchKernelGGL(orth_gram_lines_kernel<false>, dim3(gb), dim3(256), 0, st, ga);
      AGX_LAUNCH_CHECK();
      if (!one) AGX_TRY(add_slices(ra, rb, pieces));
    }
    // matrices: 0 A, 1 P, 2 A P, 3 / 4 Q (which of the two: 3 after an odd number of steps); a launch a step: 0 / 1 A
    const int steps = std::min(phase, o->steps - k);
    float coef[3 * PHASE];
    int eA[PHASE + 1], eP[PHASE], eS[PHASE], eQ[PHASE];              // scale exponents per step
    int e1[PHASE], e3[PHASE], q1[PHASE];                             // of the running rows of a launch a step
    int32_t er[E_COUNT] = {};                                        // and of a launch a phase
    double bQ = 1.0;                                                 // |Q| <= bQ
    for (int t = 0; t < steps; ++t) {
      const float *c = o->coef + (o->n_coef == 1 ? 0 : 3 * (k + t));
      const Bounds b = bounds_of(s, c[0], c[1], c[2]);
      memcpy(coef + 3 * t, c, 3 * sizeof(float));
      const double L = s * s;
      e1[t] = exponent_for(L * L); e3[t] = exponent_for(L * b.S); q1[t] = exponent_for(bQ * L);
      if (t == 0) {
        const double N = b.next * b.next;
        const double bound[E_COUNT] = {b.P, b.P * L, b.P * L * L, b.P * b.S, b.P * b.S * L,
                                       b.P * N, b.P * N * L, b.P * N * L * L, b.P * N * b.S, b.P * N * b.S * L};
        for (int i = 0; i < E_COUNT; ++i) er[i] = exponent_for(bound[i]);
      }
      bQ *= b.P;
      eA[t] = exponent_for(s * s); eP[t] = exponent_for(b.P); eS[t] = exponent_for(b.S); eQ[t] = exponent_for(bQ);
      s = b.next;
    }
    eA[steps] = exponent_for(s * s);
    k += steps;
    const int iq = steps & 1 ? 3 : 4;
    for (int t = 0; t < (any_steps ? steps : any_phases ? 1 : 0); ++t) {
      RowsArgs ra;
      memset(&ra, 0, sizeof(ra));
      ra.more = t + 1 < steps; ra.has_q = t > 0; ra.steps = steps;
      ra.a = coef[3 * t]; ra.b = coef[3 * t + 1]; ra.c = coef[3 * t + 2];
      ra.e1 = e1[t]; ra.eS = eS[t]; ra.e3 = e3[t]; ra.q1 = q1[t];
      if (steps > 1) { ra.a2 = coef[3]; ra.b2 = coef[4]; ra.c2 = coef[5]; }
      memcpy(ra.e, er, sizeof(er));
      int blocks = 0;
      for (int i = 0; i < n; ++i) {
        const int np = jobs[i].np();
        if (by_products(i) || (np <= ROWS_PHASE && t > 0)) continue;
        RowsJob &g = ra.job[ra.n++];
        g.n = jobs[i].n();
        g.first = blocks;
        if (np == STEP_NP) {
          g.A = planes(i, t & 1, eA[t]); g.An = planes(i, t & 1 ^ 1, eA[t + 1]);
          g.Q = planes(i, t & 1 ? 3 : 4, eQ[t > 0 ? t - 1 : 0]); g.Qn = planes(i, t & 1 ? 4 : 3, eQ[t]);
          blocks += STEP_NP / ROWS * 2;
        } else {
          g.A = planes(i, 0, eA[0]); g.Qn = planes(i, iq, eQ[steps - 1]);
          blocks += np / ROWS;
        }
      }
      hipLaunchKernelGGL(orth_rows_kernel, dim3(blocks), dim3(512), 0, st, ra);
      AGX_LAUNCH_CHECK();
    }
    for (int t = 0; t < steps && any_products; ++t) {
      const int in = t & 1 ? 3 : 4, out = t & 1 ? 4 : 3, iP = t == 0 ? out : 1;   // the first step's P is Q too
      auto launch = [&](int per, auto fill) -> int {
        ChainArgs ca;
        int blocks = 0;
        ca.n = 0;
        for (int i = 0; i < n; ++i)
          for (int w = 0; w < per && by_products(i); ++w) {
            ChainJob &g = ca.job[ca.n++];
            memset(&g, 0, sizeof(g));
            g.n = jobs[i].n(); g.nt = jobs[i].np() / T; g.first = blocks; g.alpha = 1.f;
            blocks += g.nt * (g.nt + 1);
            fill(g, i, w);
          }
        hipLaunchKernelGGL(orth_chain_kernel, dim3(blocks), dim3(256), 0, st, ca);
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
    auto apply = [&](bool panel) -> int {
      ApplyArgs aa;
      aa.n = 0;
      int blocks = 0, kind = -1, groups = 0;
      auto lines_of = [&](const Job &j) { return (int)(last ? j.K() : j.kp()); };
      auto groups_of = [&](const Job &j) { return agx::cdiv(lines_of(j), 8192 / j.np()); };
      for (int i = 0; i < n; ++i) groups += panel && jobs[i].np() <= PANEL_NP ? groups_of(jobs[i]) : 0;
      aa.per = agx::cdiv(groups, agx::num_cus());
      for (int i = 0; i < n; ++i) {
        const Job &j = jobs[i];
        if ((j.np() <= PANEL_NP) != panel) continue;
        ApplyJob &g = aa.job[aa.n++];
        memset(&g, 0, sizeof(g));
        g.x = j.x; g.ldx = j.ldx; g.Q = planes(i, iq, eQ[steps - 1]); g.lines = lines_of(j);
        g.maxb = reinterpret_cast<const uint32_t *>(base[i] + lay[i].maxb);
        g.invd = first ? reinterpret_cast<const double *>(base[i] + lay[i].invd) : nullptr;
        g.rows = j.rows; g.cols = j.cols; g.tall = j.tall();
        g.dtype = j.dtype; g.e = ex; g.nb = first ? nb[i] : 0;
        if (!first) g.from = iterate(ph - 1, i, ex);
        if (last) {
          g.out = j.out; g.ldo = j.ldo; g.otype = j.dtype; g.muon = j.muon; g.decay = j.decay; g.step = j.step;
        } else {
          g.to = iterate(ph, i, exponent_for(s));
        }
        kind = first ? joined_kind(kind, g.tall, g.dtype) : ITERATE;
        g.first = blocks;
        blocks += panel ? agx::cdiv(groups_of(j), aa.per) : agx::cdiv(g.lines, T) * (last ? j.nt() : j.np() / T);
      }
      if (!blocks) return AGX_OK;
      by_kind(kind, [&](auto k) {
        if (panel) hipLaunchKernelGGL(orth_panel_kernel<decltype(k)::value>, dim3(blocks), dim3(512), PANEL_LDS, st, aa);
        else hipLaunchKernelGGL(orth_apply_kernel<decltype(k)::value>, dim3(blocks), dim3(256), 0, st, aa);
      });
      AGX_LAUNCH_CHECK();
      return AGX_OK;
    };
    AGX_TRY(apply(true));
    AGX_TRY(apply(false));
  }
  return AGX_OK;
}

// (first: number of j[0] among the caller's matrices)
int to_jobs(const agx_orth_t *j, int n, Job *out, const char *who, int first = 0) {
  AGX_CHECK_ARG(j && n >= 1 && n <= AGX_MAX_ORTH, "%s: 1 to %d matrices a call", who, AGX_MAX_ORTH);
  for (int i = 0; i < n; ++i) {
    const agx_orth_t &a = j[i];
    AGX_CHECK_ARG(a.dtype == AGX_F32 || a.dtype == AGX_BF16, "%s: matrix %d: dtype %d", who, first + i, a.dtype);
    AGX_CHECK_ARG(a.rows > 0 && a.cols > 0 && std::min(a.rows, a.cols) <= AGX_ORTH_MAX_SIDE,
                  "%s: matrix %d is %d x %d; the smaller side is at most %d", who, first + i, a.rows, a.cols, AGX_ORTH_MAX_SIDE);
    AGX_CHECK_ARG((int64_t)a.rows * agx::cdiv64(a.cols, 4) < (1LL << 30) && agx::cdiv64(a.rows, T) * agx::cdiv64(a.cols, T) < (1 << 26),
                  "%s: matrix %d is too large", who, first + i);
    AGX_CHECK_ARG(a.ldx < (1 << 23) && a.ldo < (1 << 23), "%s: matrix %d: leading dimension above 2^23", who, first + i);
    Job &b = out[i];
    b.x = a.x; b.out = a.out; b.ldx = a.ldx; b.ldo = a.ldo; b.rows = a.rows; b.cols = a.cols; b.dtype = a.dtype;
  }
  return AGX_OK;
}

int muon_jobs(const agx_muon_t *j, int n, const agx_muon_opts_t *o, Job *out, const char *who, int first = 0) {
  AGX_CHECK_ARG(j && n >= 1 && n <= AGX_MAX_ORTH, "%s: 1 to %d matrices a call", who, AGX_MAX_ORTH);
  agx_orth_t m[AGX_MAX_ORTH];
  memset(m, 0, sizeof(m));
  for (int i = 0; i < n; ++i) {
    m[i].x = j[i].g; m[i].ldx = j[i].ldg; m[i].out = j[i].w; m[i].ldo = j[i].ldw;
    m[i].rows = j[i].rows; m[i].cols = j[i].cols; m[i].dtype = AGX_F32;
  }
  AGX_TRY(to_jobs(m, n, out, who, first));
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

// (more LDS than the default limit of a launch)
int agx::orth_prepare_device() {
  for (int k = 0; k <= ITERATE; ++k) {
    const void *f = nullptr;
    by_kind(k, [&](auto kind) { f = reinterpret_cast<const void *>(&orth_panel_kernel<decltype(kind)::value>); });
    AGX_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, PANEL_LDS));
  }
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
  // (matrices of a call are worked on at once)
  auto region = [&](const void *p, int i, int64_t ld) { return agx::Region{p, j[i].rows, j[i].cols, ld, j[i].dtype == AGX_F32 ? 4 : 2}; };
  for (int i = 0; i < n; ++i)
    for (int k = 0; k < n; ++k) {
      const agx::Region out = region(j[i].out, i, j[i].ldo);
      AGX_CHECK_ARG(!agx::overlap(out, region(j[k].x, k, j[k].ldx)) && (k <= i || !agx::overlap(out, region(j[k].out, k, j[k].ldo))),
                    "%s: the result of matrix %d overlaps matrix %d or its result", who, i, k);
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

// What is checked of a step's arguments apart from the workspace, over any number of matrices
static int check_muon(const agx_muon_t *jobs, int n, const agx_muon_opts_t *o, const char *who) {
  AGX_CHECK_ARG(o, "%s: options missing", who);
  AGX_TRY(check_opts(&o->orth, who));
  AGX_CHECK_ARG(o->momentum >= 0.f && o->momentum < 1.f, "%s: momentum must be in [0, 1)", who);
  AGX_CHECK_ARG(std::isfinite(o->lr) && std::isfinite(o->weight_decay), "%s: learning rate / weight decay must be finite", who);
  AGX_CHECK_ARG(jobs && n >= 1, "%s: no matrices", who);
  Job j[AGX_MAX_ORTH];
  for (int lo = 0; lo < n; lo += AGX_MAX_ORTH) AGX_TRY(muon_jobs(jobs + lo, std::min(n - lo, AGX_MAX_ORTH), o, j, who, lo));
  for (int i = 0; i < n; ++i) {
    const agx_muon_t &a = jobs[i];
    AGX_CHECK_ARG(a.w && a.g && a.m && a.ldw >= a.cols && a.ldg >= a.cols && a.ldm >= a.cols && a.ldm < (1 << 23) && std::isfinite(a.scale),
                  "%s: matrix %d: null, leading dimension or scale", who, i);
    AGX_CHECK_ARG(((reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.g) | reinterpret_cast<uintptr_t>(a.m)) & 3) == 0,
                  "%s: matrix %d not aligned to its elements", who, i);
    AGX_CHECK_ARG(a.w != a.m && a.w != a.g && a.g != a.m, "%s: matrix %d: w, g and m must be different arrays", who, i);
  }
  // (matrices of a call are worked on at once: what is written, w and m, must be nothing else's)
  auto region = [&](const void *p, int i, int64_t ld) { return agx::Region{p, jobs[i].rows, jobs[i].cols, ld, 4}; };
  for (int i = 0; i < n; ++i)
    for (int k = 0; k < n; ++k) {
      const agx::Region w = region(jobs[i].w, i, jobs[i].ldw), m = region(jobs[i].m, i, jobs[i].ldm), g = region(jobs[k].g, k, jobs[k].ldg);
      const agx::Region wk = region(jobs[k].w, k, jobs[k].ldw), mk = region(jobs[k].m, k, jobs[k].ldm);
      AGX_CHECK_ARG(!agx::overlap(w, g) && !agx::overlap(m, g) && !agx::overlap(w, mk) && (k <= i || (!agx::overlap(w, wk) && !agx::overlap(m, mk))),
                    "%s: w, g and m of matrices %d and %d must be different arrays", who, std::min(i, k), std::max(i, k));
    }
  return AGX_OK;
}

extern "C" int agx_opt_muon_check(const agx_muon_t *jobs, int32_t n, const agx_muon_opts_t *o) {
  return check_muon(jobs, n, o, "agx_opt_muon_check");
}

extern "C" int agx_opt_muon(void *stream, const agx_muon_t *jobs, int32_t n, const agx_muon_opts_t *o, void *ws, int64_t ws_size) {
  const char *who = "agx_opt_muon";
  AGX_CHECK_ARG(n <= AGX_MAX_ORTH, "%s: 1 to %d matrices a call", who, AGX_MAX_ORTH);
  AGX_TRY(check_muon(jobs, n, o, who));
  Job j[AGX_MAX_ORTH];
  AGX_TRY(muon_jobs(jobs, n, o, j, who));
  return run(agx::as_stream(stream), j, n, &o->orth, o->momentum, o->nesterov != 0, static_cast<char *>(ws), ws_size, who);
}
