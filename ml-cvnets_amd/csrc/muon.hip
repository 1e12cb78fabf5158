// Orthogonalised updates: Newton-Schulz products on a list of matrices, and the optimizer step around them.
//
//   u = g  (orthogonalize)   or   mom <- mu mom + g,  u = g + mu mom (Nesterov) or mom  (optimizer step)
//   x <- u / (|u|_F + eps), the shorter side m as rows;   `steps` times:  G = x x^T,  P = b G + c G G,  x <- a x + P x
//   result = x   or   w <- (1 - lr wd) w - lr gain x
//
// G and P are symmetric and commute: half of their tiles are computed and written twice.  Operands are kept as pairs of fp16 numbers, hi + lo,
// of the value times a power of two (x: 2^12, so that singular values below 16 stay under fp16's 65504 and an entry of ordinary size far above its
// subnormals; G and P: 2^12 and 2^10, or what the coefficients leave room for, see Bounds): 22 bits and a sign, and a product is three MFMAs, hi hi + hi lo + lo hi, accumulated in float32 -
// results as near to the exact ones as those of float32 products (from 41 rows on, see few rows), at a third of the fp16 matrix rate instead of the float32 matrix rate (measured on 8192-cubed library products: 1081 / 3
// = 360 against 154 TFLOP/s).  One fp16 or bf16 product per step would be three times as fast, and its rounding (2^-11 and 2^-8) is multiplied by up to
// a^steps = 485 in the directions of small singular values.
//
// (a x is added to the finished sum: with a I inside P the small terms of the long sum are rounded next to a x, 8e-6 instead of 2e-6 after 5
// steps of a 1030 x 1100 matrix, whose float32 products give 2e-6, too.)
// x is kept once, [m][n] (contraction over n: rows times rows); P x reads its columns with LDS transpose reads.  The cross products hi lo + lo hi
// have accumulators of their own: the large sum is then rounded once per 16 terms instead of three times.  Every epilogue goes through
// LDS, so that global memory sees whole rows.  Sides are padded to the tile with zeros, which the products keep zero: the main loop has no bounds.
// All matrices of a list go through one launch per product: 2 + 3 steps launches for up to kMats matrices.
//
// Measured: 24 matrices of a 6-layer text tower of 512 (1536 x 512 .. 512 x 2048, float32): 830 .. 900 us (cards differ), of 526 at the library's rates; 4096 x 2048 in
// bf16: 1175 .. 1280 of 842 us (P x at 880 TFLOP/s of MFMA; x x^T has 136 tiles for 256 units); 21 matrices of 144 .. 720: 161 us, 17 dependent launches of 7 .. 14 us.
#include "common.hpp"
#include "cvnets_hip.h"

namespace {

constexpr int kMats = 32;
constexpr int kMostRows = 1 << 14, kMostCols = 1 << 20;  // of the shorter and the longer side
constexpr float kScale = 4096.f;  // of x
typedef _Float16 half_t;
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

struct Mat {
  const void* src;  // u, or the gradient (float32)
  void* dst;        // result (orthogonalize)
  float *mom, *par;
  half_t* ws;       // x [mp][2 np] twice (ping-pong), G [mp][2 mp], P [mp][2 mp]; see place()
  double* norm;     // partial sums of squares
  int m, n, mp, np, rows, cols, group;
  float gain;
};
// The list: an argument of the first kernel, which leaves a copy in the workspace for the others (arguments lie in host memory: a workgroup's two
// dependent reads of them cost more than a small matrix's product).
enum { NORM, SCALE, SYM, APPLY, PHASES };
struct Mats {
  Mat mat[kMats];
  int first[PHASES][kMats + 1];  // prefixes of workgroups; behind the last matrix: their number
  int count, steps, nesterov;
  float a, b, c, eps, mu;
};
// the matrix that workgroup `wg` of a phase works on, for all of its waves: lane i compares the end of matrix i
__device__ __forceinline__ int find(const Mats& t, int phase, int wg) {
  const int lane = threadIdx.x & 63;
  return __popcll(__ballot(lane < kMats && wg >= t.first[phase][min(lane, kMats - 1) + 1]));
}
// Pointers that were loaded from memory have no address space, and accesses through them would be flat ones, which count as LDS instructions, too
// (10 % of the products' time): they are cast to global ones.
#define GLOBAL __attribute__((address_space(1)))
typedef GLOBAL half_t ghalf_t;
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
template <typename V> __device__ __forceinline__ V gload(const ghalf_t* p) { return *(const GLOBAL V*)p; }
template <typename V> __device__ __forceinline__ void gstore(ghalf_t* p, V v) { *(GLOBAL V*)p = v; }
template <typename T> __device__ __forceinline__ float gvalue(const void* p, size_t i) {
  if constexpr (sizeof(T) == 4) return ((const GLOBAL float*)p)[i];
  else return bf2f(((const GLOBAL uint16_t*)p)[i]);
}
template <typename T> __device__ __forceinline__ void gput(void* p, size_t i, float v) {
  if constexpr (sizeof(T) == 4) ((GLOBAL float*)p)[i] = v;
  else ((GLOBAL uint16_t*)p)[i] = f2bf(v);
}
__device__ __forceinline__ size_t plane_x(const Mat& a) { return (size_t)a.mp * a.np; }
__device__ __forceinline__ ghalf_t* x_of(const Mat& a, int which) { return (ghalf_t*)a.ws + (size_t)which * 2 * plane_x(a); }
__device__ __forceinline__ ghalf_t* g_of(const Mat& a) { return (ghalf_t*)a.ws + 4 * plane_x(a); }
__device__ __forceinline__ ghalf_t* p_of(const Mat& a) { return g_of(a) + 2 * (size_t)a.mp * a.mp; }

// A row of pairs is in blocks of 32 columns, 32 hi and then their 32 lo: one 128-byte line.  A step of 32 columns of the products reads whole lines;
// with the two halves in matrices of their own it reads half lines, each of them twice.  place(): of the hi of 8 columns; lo is kLo behind it.
constexpr int kLo = 32;
__device__ __forceinline__ size_t place(int row, int col, int ld) { return (size_t)row * 2 * ld + (col >> 5) * 64 + (col & 31); }

__device__ __forceinline__ void split(float v, half_t& hi, half_t& lo) {
  hi = (half_t)v;
  lo = (half_t)(v - (float)hi);
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// sums of squares (and the momentum), kNormItems elements a workgroup; in 64 bits, so that no gradient's square leaves the range
// -----------------------------------------------------------------------------------------------------------------------------------------
constexpr int kNormItems = 8192;
template <typename T, bool MOM> __device__ __forceinline__ float update_of(const Mat& a, size_t i, float mu, int nesterov) {
  const float g = gvalue<T>(a.src, i);
  if (!MOM) return g;
  const float m = gvalue<float>(a.mom, i);
  return nesterov ? g + mu * m : m;
}
template <typename T, bool MOM> __global__ __launch_bounds__(256) void ns_norm_kernel(Mats t, Mats* copy, float mu, int nesterov) {
  __shared__ double sums[4];
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < (int)(sizeof(Mats) / 4); i += 256) reinterpret_cast<int*>(copy)[i] = reinterpret_cast<const int*>(&t)[i];
  const int k = find(t, NORM, blockIdx.x), chunk = blockIdx.x - t.first[NORM][k];
  const Mat& a = t.mat[k];
  const size_t size = (size_t)a.m * a.n, i0 = (size_t)chunk * kNormItems, i1 = i0 + kNormItems < size ? i0 + kNormItems : size;
  const T* const src = reinterpret_cast<const T*>(a.src);
  double s = 0.0;
  auto one = [&](float g, float m) {
    const double u = MOM ? (nesterov ? g + mu * m : m) : g;
    s += u * u;
  };
  size_t done = i0;
  if (((reinterpret_cast<uintptr_t>(src) | (MOM ? reinterpret_cast<uintptr_t>(a.mom) : 0)) & 15) == 0) {
    done = i0 + (i1 - i0) / 4 * 4;
    for (size_t i = i0 + threadIdx.x * 4; i < done; i += 1024) {
      float g[4], m[4] = {0.f, 0.f, 0.f, 0.f};
      v4_unpack(v4_load<T>(src + i), g);
      if (MOM) {
        v4_unpack(v4_load<float>(a.mom + i), m);
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = mu * m[e] + g[e];
        *reinterpret_cast<float4*>(a.mom + i) = make_float4(m[0], m[1], m[2], m[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) one(g[e], m[e]);
    }
  }
  for (size_t i = done + threadIdx.x; i < i1; i += 256) {
    const float g = to_f<T>(src[i]);
    float m = 0.f;
    if (MOM) a.mom[i] = m = mu * a.mom[i] + g;
    one(g, m);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.norm[chunk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// Matrices of few rows.  All steps are one polynomial of u u^T, and with few rows that is small enough for 64 bits: G = u u^T from partial sums (in the
// scale kernel), Q = the product of the steps' a I + b G + c G^2, G <- (..) G (..) (one workgroup, in the first launch for x x^T), result = Q u / (|u| + eps)
// (in the first launch of P x): no launch more, and none behind the first step where all matrices of a list are such.  Not for speed: one singular direction
// is a large part of such a matrix, and pairs of 22 bits through five steps leave an error that nothing averages: 1 .. 16 rows 0.8 .. 1.7e-6 where float32
// products leave 0.5 .. 1.1e-6, now 0.4 .. 0.6e-7; from 40 rows on the pairs leave 0.7 .. 1.5e-6 where those leave 0.8 .. 3.1e-6.  (In the chain of
// products / so: 1 x 640 86 / 24 us, 16 x 2500 160 / 31, 40 x 40 63 / 57, 40 x 100000 3765 / 198; eight 16 x 144 next to eight 192 x 576 130 / 133.)
// In the workspace: partial sums [chunk][pair i >= j], then Q.
// -----------------------------------------------------------------------------------------------------------------------------------------
constexpr int kFewRows = 40, kFewCols = 64, kFewChunks = 256;  // columns of a workgroup of the result; most chunks of the partial sums, 64 columns and more each
typedef GLOBAL double gdouble_t;
__host__ __device__ __forceinline__ bool few(const Mat& a) { return a.m <= kFewRows; }
__host__ __device__ __forceinline__ int few_chunks(const Mat& a) { return a.n < 64 * kFewChunks ? (a.n + 63) / 64 : kFewChunks; }
__device__ __forceinline__ int pairs_of(int m) { return m * (m + 1) / 2; }
__device__ __forceinline__ gdouble_t* few_parts(const Mat& a) { return (gdouble_t*)a.ws; }
__device__ __forceinline__ gdouble_t* few_q(const Mat& a) { return few_parts(a) + (size_t)few_chunks(a) * pairs_of(a.m); }
__device__ __forceinline__ void pair_at(int p, int& i, int& j) {
  for (i = 0; p > i; ++i) p -= i + 1;
  j = p;
}

template <typename T, bool MOM> __device__ __forceinline__ void few_gram(const Mat& a, int chunk, float (*tile)[65], double* red, float mu, int nesterov) {
  constexpr int MOST = (kFewRows * (kFewRows + 1) / 2 + 255) / 256, LOADS = 5;  // pairs of a thread, elements that it loads at a time
  const int tid = threadIdx.x, m = a.m, n = a.n, pairs = pairs_of(m), chunks = few_chunks(a);
  const int per = ((n + chunks - 1) / chunks + 63) & ~63, c0 = chunk * per, c1 = min(c0 + per, n);
  int slices = 1;  // of the columns, where there are fewer pairs than threads
  while (slices * 2 * pairs <= 256) slices *= 2;
  const bool narrow = pairs <= 256;
  const int mine = narrow ? tid % pairs : tid, slice = narrow ? tid / pairs : 0;
  int pi[MOST], pj[MOST];
  double sum[MOST];
#pragma unroll
  for (int q = 0; q < MOST; ++q) {
    pair_at(mine + 256 * q < pairs ? mine + 256 * q : 0, pi[q], pj[q]);
    sum[q] = 0.0;
  }
  const bool flip = a.rows > a.cols;
  for (int c = c0; c < c1; c += 64) {
#pragma unroll 1
    for (int base = tid; base < 64 * m; base += 256 * LOADS) {
      float v[LOADS];  // in flight together (what is not there: the first element)
#pragma unroll
      for (int q = 0; q < LOADS; ++q) {
        const int idx = base + 256 * q, i = flip ? idx % m : idx >> 6, j = flip ? idx / m : idx & 63;
        const bool here = idx < 64 * m && c + j < c1;
        v[q] = update_of<T, MOM>(a, !here ? 0 : flip ? (size_t)(c + j) * m + i : (size_t)i * n + c + j, mu, nesterov);
        v[q] = here ? v[q] : 0.f;
      }
#pragma unroll
      for (int q = 0; q < LOADS; ++q) {
        const int idx = base + 256 * q;
        if (idx < 64 * m) tile[flip ? idx % m : idx >> 6][flip ? idx / m : idx & 63] = v[q];
      }
    }
    __syncthreads();
    if (slice < slices) {
#pragma unroll
      for (int q = 0; q < MOST; ++q) {
        if (q > 0 && 256 * q >= pairs) continue;
        const float *x = tile[pi[q]], *y = tile[pj[q]];
#pragma unroll 4
        for (int k = slice; k < 64; k += slices) sum[q] += (double)x[k] * (double)y[k];
      }
    }
    __syncthreads();
  }
  gdouble_t* const out = few_parts(a) + (size_t)chunk * pairs;
  if (narrow) {
    red[tid] = sum[0];
    __syncthreads();
    if (tid < pairs) {
      double s = 0.0;
      for (int k = 0; k < slices; ++k) s += red[k * pairs + tid];
      out[tid] = s;
    }
  } else {
#pragma unroll
    for (int q = 0; q < MOST; ++q)
      if (tid + 256 * q < pairs) out[tid + 256 * q] = sum[q];
  }
}

// Q by one workgroup.  G, Q and the matrices between them are polynomials of one symmetric matrix: they commute, and their products are symmetric; 2 x 2
// elements at or below the diagonal a thread, rows and columns up to a multiple of 4 stay zero.  Reading the LDS bounds it (4 x 4 elements a thread: half the
// reads, but half of the card's units for doubles of this workgroup idle, and slower).
constexpr size_t kFewBytes = 3 * sizeof(double) * kFewRows * (kFewRows + 2);
__device__ __forceinline__ void few_solve(const Mats& t, const Mat& a, double* lds) {
  static_assert(kFewRows % 4 == 0 && kFewRows / 2 * (kFewRows / 2 + 1) / 2 <= 256, "a square of a product a thread");
  const int tid = threadIdx.x, m = a.m, size = (m + 3) & ~3, half = size / 2, ld = size + 2, pairs = pairs_of(m), chunks = few_chunks(a);
  double *const G = lds, *const Q = G + size * ld, *const M = Q + size * ld;
  for (int i = tid; i < 3 * size * ld; i += 256) lds[i] = 0.0;
  __syncthreads();
  const gdouble_t* const parts = few_parts(a);
  for (int p = tid; p < pairs; p += 256) {
    double s = 0.0;
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) s += parts[(size_t)c * pairs + p];
    int i, j;
    pair_at(p, i, j);
    G[i * ld + j] = G[j * ld + i] = s;
  }
  if (tid < m) Q[tid * ld + tid] = 1.0;
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < m; ++i) total += G[i * ld + i];
  const double inv = 1.0 / (sqrt(total) + (double)t.eps);
  __syncthreads();
  for (int i = tid; i < size * ld; i += 256) G[i] *= inv * inv;
  __syncthreads();
  const bool in = tid < half * (half + 1) / 2;
  int i0, j0;
  pair_at(in ? tid : 0, i0, j0);
  i0 *= 2;
  j0 *= 2;
  struct Out {
    double v[2][2];
  };
  auto multiply = [&](const double* A, const double* B) {
    Out o = {};
    if (!in) return o;
    for (int k = 0; k < size; k += 4) {
      double x[4][2], y[4][2];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          x[e][f] = A[(i0 + f) * ld + k + e];
          y[e][f] = B[(k + e) * ld + j0 + f];
        }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) o.v[r][c] += x[e][r] * y[e][c];
    }
    return o;
  };
  auto put = [&](double* D, const Out& o) {  // (a square on the diagonal: its lower three)
    if (!in) return;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (j0 + c <= i0 + r) D[(i0 + r) * ld + j0 + c] = D[(j0 + c) * ld + i0 + r] = o.v[r][c];
  };
  for (int s = 0; s < t.steps; ++s) {
    Out o = multiply(G, G);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const double g = in ? G[(i0 + r) * ld + j0 + c] : 0.0;
        o.v[r][c] = (i0 + r == j0 + c && i0 + r < m ? (double)t.a : 0.0) + (double)t.b * g + (double)t.c * o.v[r][c];
      }
    put(M, o);
    __syncthreads();
    if (s > 0) o = multiply(M, Q);  // (Q is one)
    if (s + 1 == t.steps) {
      __syncthreads();
      put(Q, o);
      break;
    }
    const Out w = multiply(M, G);
    __syncthreads();
    put(Q, o);
    put(G, w);
    __syncthreads();
    o = multiply(G, M);
    __syncthreads();
    put(G, o);
    __syncthreads();
  }
  __syncthreads();
  gdouble_t* const out = few_q(a);
  for (int i = tid; i < m * m; i += 256) out[i] = Q[i / m * ld + i % m] * inv;
}

// result = Q u: 64 columns, a lane a column, the rows dealt out to the four waves
template <typename T> __device__ __forceinline__ void few_apply(const Mats& t, const Mat& a, int part, double* lds, const float* __restrict__ hp) {
  const int tid = threadIdx.x, m = a.m, n = a.n, j = part * kFewCols + (tid & 63);
  const bool flip = a.rows > a.cols;
  auto place_of = [&](int i) { return flip ? (size_t)min(j, n - 1) * m + i : (size_t)i * n + min(j, n - 1); };
  double u[kFewRows];
#pragma unroll
  for (int k = 0; k < kFewRows; ++k) {
    const size_t at = place_of(min(k, m - 1));  // (all loads in flight)
    u[k] = k < m ? (double)(a.mom != nullptr ? update_of<float, true>(a, at, t.mu, t.nesterov) : update_of<T, false>(a, at, 0.f, 0)) : 0.0;
  }
  const gdouble_t* const q = few_q(a);
#pragma unroll 4
  for (int i = tid; i < m * kFewRows; i += 256) {
    const double v = q[i / kFewRows * m + min(i % kFewRows, m - 1)];
    lds[i] = i % kFewRows < m ? v : 0.0;
  }
  __syncthreads();  // (u is read: the result may be written over it)
  if (j >= n) return;
  const float lr = a.par != nullptr ? hp[2 * a.group] : 0.f, keep = a.par != nullptr ? 1.f - lr * hp[2 * a.group + 1] : 0.f, step = lr * a.gain;
  for (int i = tid >> 6; i < m; i += 4) {
    const float old = a.par != nullptr ? gvalue<float>(a.par, place_of(i)) : 0.f;
    double y[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int k = 0; k < kFewRows; ++k) y[k & 3] += lds[i * kFewRows + k] * u[k];
    const float v = (float)((y[0] + y[1]) + (y[2] + y[3]));
    if (a.par != nullptr) gput<float>(a.par, place_of(i), old * keep - step * v);
    else gput<T>(a.dst, place_of(i), v);
  }
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// x = u / (|u| + eps), 64 x 64 elements (of the padded matrix) a workgroup; through LDS where the matrix is taller than wide
// -----------------------------------------------------------------------------------------------------------------------------------------
template <typename T, bool MOM> __global__ __launch_bounds__(256) void ns_scale_kernel(const Mats* __restrict__ list, float mu, int nesterov, float eps) {
  const Mats& t = *list;
  __shared__ float tile[64][65];
  __shared__ double total, red[256];
  const int k = find(t, SCALE, blockIdx.x), at = blockIdx.x - t.first[SCALE][k], tid = threadIdx.x;
  const Mat& a = t.mat[k];
  if (few(a)) {
    few_gram<T, MOM>(a, at, tile, red, mu, nesterov);
    return;
  }
  const int tn = a.np / 64, i0 = at / tn * 64, j0 = at % tn * 64;
  const bool flip = a.rows > a.cols;  // x[i][j] = u[j][i]
  float v[16];
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int r = q * 4 + (tid >> 6), c = tid & 63;  // of u's tile: c runs along u's rows
    const int i = flip ? i0 + c : i0 + r, j = flip ? j0 + r : j0 + c;
    v[q] = i < a.m && j < a.n ? update_of<T, MOM>(a, (size_t)(flip ? j : i) * a.cols + (flip ? i : j), mu, nesterov) : 0.f;
  }
  if (tid < 64) {
    const int chunks = (int)(((size_t)a.m * a.n + kNormItems - 1) / kNormItems);
    double s = 0.0;
    for (int c = tid; c < chunks; c += 64) s += ((const GLOBAL double*)a.norm)[c];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (tid == 0) total = s;
  }
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int r = q * 4 + (tid >> 6), c = tid & 63;
    if (flip) tile[c][r] = v[q]; else tile[r][c] = v[q];
  }
  __syncthreads();
  const double inv = (double)kScale / (sqrt(total) + (double)eps);
  ghalf_t* const x = x_of(a, 0);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = q * 16 + (tid >> 4), c = (tid & 15) * 4;
    half4_t hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      half_t h, l;
      split((float)(tile[r][c + e] * inv), h, l);
      hi[e] = h;
      lo[e] = l;
    }
    const size_t o = place(i0 + r, j0 + c, a.np);
    gstore(x + o, hi);
    gstore(x + o + kLo, lo);
  }
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// product of hi + lo operands on a TR x TC tile by WAVES waves: acc[r][c] = sum_k A[r][k] B[c][k], B in rows; A in rows, or (COLS) given as
// [k][r] and read with LDS transpose reads.  Two LDS stages of BK.  First half of step t: its second 16-wide slice is read and its first one multiplied;
// barrier: its stage is free and step t + 1's complete; second half: t + 2 goes from registers (requested a step and a half before) into the free stage,
// and the first slice of t + 1 is read under t's last MFMAs.  With reads and MFMAs of a slice in sequence the time was their sum, whatever the depth
// of the global prefetch.  The lo halves lie 16 banks off the hi halves (+ 32): eight lanes of a write, a global line of 32 hi and 32 lo, hit 32 banks
// instead of 16 twice (with the pitch of the transpose reads: LDS conflicts from 30 % of its busy cycles to 0, the products 1 .. 4 % faster).
// 4096 x 2048: MFMA busy in 61 % of the cycles in x x^T, 53 % in P x, at 2.0 .. 2.1 GHz (the library's large product reaches 43 % of the peak).
// -----------------------------------------------------------------------------------------------------------------------------------------
typedef short v4s_t __attribute__((ext_vector_type(4)));
template <int TR, int TC, int WAVES, bool COLS> struct Product {
  static constexpr int NT = 64 * WAVES, BK = 32, PITCH = BK + 8;  // rows of 80 bytes: 16 lanes' 16-byte reads hit distinct banks
  static constexpr int WR = TR * 2 / WAVES, WC = TC / 2;  // rows and columns of a wave
  static constexpr int FR = WR / 32, FC = WC / 32;            // 32-wide fragments of them
  static constexpr int CA = 8 * TR / NT, CB = 8 * TC / NT;    // 16-byte pieces a thread loads of each operand
  static constexpr int CPITCH = TR + 32;                      // [k][r] rows: the 4 rows of a transpose read are 16 banks apart
  static constexpr int AELEMS = (COLS ? BK * CPITCH : TR * PITCH) + 32, BELEMS = TC * PITCH + 32, STAGE = 2 * AELEMS + 2 * BELEMS;
  static constexpr int OPITCH = TR + 4;                     // of the float tile of the epilogue
  static constexpr size_t BYTES = sizeof(half_t) * 2 * STAGE > sizeof(float) * TC * OPITCH ? sizeof(half_t) * 2 * STAGE : sizeof(float) * TC * OPITCH;
  half_t* lds;
  f32x16_t acc[FR][FC];
  u32x4_t qa[2][CA], qb[2][CB];
  struct Frags {
    half8_t ah[FR], al[FR], bh[FC], bl[FC];
  };

  static __device__ __forceinline__ int row0(int tid) { return (tid >> 7) * WR; }
  static __device__ __forceinline__ int col0(int tid) { return ((tid >> 6) & 1) * WC; }
  // pieces of 16 bytes, in the order of the global lines: row r = 4 hi and 4 lo pieces (COLS: row k = TILE / 4 pieces)
  template <int S> __device__ __forceinline__ void load(const ghalf_t* a, int lda, const ghalf_t* b, int ldb, int k0, int tid) {
#pragma unroll
    for (int c = 0; c < CA; ++c) {
      const int idx = tid + c * NT, r = idx >> 3, in = (idx & 7) * 8;
      qa[S][c] = gload<u32x4_t>(COLS ? a + (size_t)(k0 + idx / (TR / 4)) * 2 * lda + idx % (TR / 4) * 8 : a + (size_t)r * 2 * lda + k0 * 2 + in);
    }
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const int idx = tid + c * NT;
      qb[S][c] = gload<u32x4_t>(b + (size_t)(idx >> 3) * 2 * ldb + k0 * 2 + (idx & 7) * 8);
    }
  }
  template <int S> __device__ __forceinline__ void store(int stage, int tid) {
    half_t* const s = lds + stage * STAGE;
    auto rows = [&](int idx) { return (idx >> 3) * PITCH + (idx & 3) * 8; };
#pragma unroll
    for (int c = 0; c < CA; ++c) {
      const int idx = tid + c * NT, in = idx % (TR / 4);
      *reinterpret_cast<u32x4_t*>(s + ((idx >> 2) & 1) * AELEMS + (COLS ? idx / (TR / 4) * CPITCH + (in >> 3) * 32 + (idx & 3) * 8 : rows(idx))) = qa[S][c];
    }
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const int idx = tid + c * NT;
      *reinterpret_cast<u32x4_t*>(s + 2 * AELEMS + ((idx >> 2) & 1) * BELEMS + rows(idx)) = qb[S][c];
    }
  }
  static __device__ __forceinline__ half8_t row_frag(const half_t* t, int row, int k, int lane) {
    return *reinterpret_cast<const half8_t*>(t + (row + (lane & 31)) * PITCH + k + 8 * (lane >> 5));
  }
  static __device__ __forceinline__ half8_t col_frag(const half_t* t, int row, int k, int lane) {
    const int i = lane & 15;
    const half_t* p = t + (k + 8 * (lane >> 5) + (i >> 2)) * CPITCH + row + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
    const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_t*)(p));
    const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_t*)(p + 4 * CPITCH));
    return __builtin_bit_cast(half8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // order of the instructions since the last call: LDS reads, and the four instructions of class OTHER (LDS writes 0x200, global loads 0x020), between the MFMAs
  template <int OTHER> static __device__ __forceinline__ void interleave() {
    constexpr int MFMAS = 3 * FR * FC, READS = (COLS ? 4 : 2) * FR + 2 * FC, OTHERS = CA + CB;
    static_for<0, MFMAS>([](auto i) {
      constexpr int r = (i + 1) * READS / MFMAS - i * READS / MFMAS, o = (i + 1) * OTHERS / MFMAS - i * OTHERS / MFMAS;
      if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if constexpr (o > 0) __builtin_amdgcn_sched_group_barrier(OTHER, o, 0);
    });
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void run(const ghalf_t* a, int lda, const ghalf_t* b, int ldb, int K, int tid) {
    const int lane = tid & 63, wr = row0(tid), wc = col0(tid);
    f32x16_t cross[FR][FC];
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int j = 0; j < FC; ++j) acc[i][j] = cross[i][j] = acc_zero();
    const int steps = K / BK;
    auto request = [&](auto set, int t) { this->template load<decltype(set)::value>(a, lda, b, ldb, t * BK, tid); };
    auto read = [&](int stage, int k) {
      const half_t* const st = lds + stage * STAGE;
      Frags f;
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        f.ah[i] = COLS ? col_frag(st, wr + 32 * i, k, lane) : row_frag(st, wr + 32 * i, k, lane);
        f.al[i] = COLS ? col_frag(st + AELEMS, wr + 32 * i, k, lane) : row_frag(st + AELEMS, wr + 32 * i, k, lane);
      }
#pragma unroll
      for (int j = 0; j < FC; ++j) {
        f.bh[j] = row_frag(st + 2 * AELEMS, wc + 32 * j, k, lane);
        f.bl[j] = row_frag(st + 2 * AELEMS + BELEMS, wc + 32 * j, k, lane);
      }
      return f;
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j) {
          cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[i], f.bh[j], cross[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bh[j], acc[i][j], 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j) cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bl[j], cross[i][j], 0, 0, 0);
    };
    typedef std::integral_constant<int, 0> S0;
    typedef std::integral_constant<int, 1> S1;
    // No branch inside the loop (steps is even: sides are multiples of 64): behind one the compiler's counts of outstanding loads are
    // lower bounds and every wait becomes a wait for the newest load.  Steps past the end load the last one again, into stages nobody reads.
    request(S0{}, 0);
    request(S1{}, 1);
    this->template store<0>(0, tid);
    request(S0{}, min(2, steps - 1));
    this->template store<1>(1, tid);
    wg_barrier_lds();
    Frags f = read(0, 0);
    for (int t0 = 0; t0 < steps; t0 += 2)
      static_for<0, 2>([&](auto d) {
        // A wave that issues its LDS instructions in a row waits for the LDS queue with its MFMAs behind it, as the other waves do at the same
        // time, and the LDS is idle while they all multiply: one LDS instruction between two MFMAs keeps both busy.
        constexpr int D = decltype(d)::value;
        Frags next;
        request(std::integral_constant<int, 1 - D>{}, min(t0 + D + 3, steps - 1));
        next = read(D, 16);
        multiply(f);
        interleave<0x020>();
        f = next;
        wg_barrier_lds();
        this->template store<D>(D, tid);
        next = read(1 - D, 0);
        multiply(f);
        interleave<0x200>();
        f = next;
      });
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int j = 0; j < FC; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] += cross[i][j][r];
  }
  // the tile as floats in LDS, transposed: out[c][r]
  __device__ __forceinline__ float* spill(int tid) {
    const int lane = tid & 63, wr = row0(tid), wc = col0(tid);
    float* const out = reinterpret_cast<float*>(lds);
    __syncthreads();  // the operands are read
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int j = 0; j < FC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<float4*>(out + (wc + 32 * j + (lane & 31)) * OPITCH + wr + 32 * i + 8 * e + 4 * (lane >> 5)) =
              make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]);
    __syncthreads();
    return out;
  }
};

__device__ __forceinline__ void split8(const float* v, half8_t& hi, half8_t& lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    half_t h, l;
    split(v[e], h, l);
    hi[e] = h;
    lo[e] = l;
  }
}
// Tiles are numbered in squares of 4 x 4, and 16 consecutive ones run on one XCD (block b runs on XCD b % 8): they read 8 operand panels instead of
// 32 into that XCD's L2, which the whole operand (4096 x 2048: 34 MB) does not fit.  In row order the products ran at the rate of the memory-side cache.
__device__ __forceinline__ int near_tiles(int b, int n) {
  const int whole = n & ~127;
  if (b < whole) return (b & ~127) + (b & 7) * 16 + ((b & 127) >> 3);
  const int r = b - whole, some = (n - whole) & ~31;
  return whole + (r < some ? (r & ~31) + (r & 7) * 4 + ((r & 31) >> 3) : r);
}
// tile `at` of an nr x nc grid in that order: squares column by column, each column by column
__device__ __forceinline__ void square_tile(int at, int nr, int nc, int& i, int& j) {
  const int strip = at / (4 * nr), in = at - strip * 4 * nr, w = min(4, nc - strip * 4);  // a strip is 4 (the last one w) columns
  const int band = in / (4 * w), r = in - band * 4 * w, h = min(4, nr - band * 4);
  i = band * 4 + r % h;
  j = strip * 4 + r / h;
}
// tile `at` of the lower triangle (j <= i) of an n x n grid: squares row by row, those on the diagonal being triangles themselves
__device__ __forceinline__ void triangle_tile(int at, int n, int& i, int& j) {
  int band = 0;
  for (;; ++band) {  // band of 4 (the last one h) rows: 4 h tiles a square and a triangle
    const int h = min(4, n - band * 4), size = 4 * h * band + h * (h + 1) / 2;
    if (at < size) {
      if (at < 4 * h * band) {
        const int r = at % (4 * h);
        i = band * 4 + r % h;
        j = at / (4 * h) * 4 + r / h;
      } else {
        at -= 4 * h * band;
        int ti = 0;
        while (at > ti) at -= ++ti;
        i = band * 4 + ti;
        j = band * 4 + at;
      }
      return;
    }
    at -= size;
  }
}

// G = x x^T (POLY false) or P = b G + c G G (true): tiles (i, j <= i), written to both halves.  scale_g, scale_p: what G and P are stored times.
template <int TILE, int WAVES, bool POLY>
__global__ __launch_bounds__(64 * WAVES, 2) void ns_sym_kernel(const Mats* __restrict__ list, int step, float cb, float cc, float scale_g, float scale_p) {
  const Mats& t = *list;
  typedef Product<TILE, TILE, WAVES, false> Prod;
  __shared__ __attribute__((aligned(16))) char smem[Prod::BYTES];
  const int block = near_tiles(blockIdx.x, gridDim.x), k = find(t, SYM, block), tid = threadIdx.x, which = step & 1;
  const Mat a = t.mat[k];
  if constexpr (TILE == 64) {  // (a list with such a matrix takes the small tiles: its sides are not multiples of 128)
    static_assert(Prod::BYTES >= kFewBytes, "three matrices of doubles");
    if (few(a)) {
      if (!POLY && step == 0) few_solve(t, a, reinterpret_cast<double*>(smem));
      return;
    }
  }
  int ti, tj;
  triangle_tile(block - t.first[SYM][k], a.mp / TILE, ti, tj);
  const int i0 = ti * TILE, j0 = tj * TILE;
  ghalf_t* const g = g_of(a);
  Prod p;
  p.lds = reinterpret_cast<half_t*>(smem);
  if (POLY) p.run(g + place(i0, 0, a.mp), a.mp, g + place(j0, 0, a.mp), a.mp, a.mp, tid);
  else p.run(x_of(a, which) + place(i0, 0, a.np), a.np, x_of(a, which) + place(j0, 0, a.np), a.np, a.np, tid);
  ghalf_t* const out = POLY ? p_of(a) : g;
  constexpr int PIECES = TILE * TILE / 8 / Prod::NT;
  half8_t gh[PIECES], gl[PIECES];
  if (POLY) {
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int idx = tid + q * Prod::NT;
      const size_t o = place(j0 + idx / (TILE / 8), i0 + idx % (TILE / 8) * 8, a.mp);
      gh[q] = gload<half8_t>(g + o);
      gl[q] = gload<half8_t>(g + o + kLo);
    }
  }
  float* const v = p.spill(tid);  // v[j][i]
  const float unscale = POLY ? 1.f / scale_g : scale_g / (kScale * kScale), rescale = scale_p / scale_g;  // (powers of two: exact)
#pragma unroll
  for (int q = 0; q < PIECES; ++q) {
    const int idx = tid + q * Prod::NT, j = idx / (TILE / 8), i = idx % (TILE / 8) * 8;
    const size_t o = place(j0 + j, i0 + i, a.mp);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v[j * Prod::OPITCH + i + e] * unscale;
    if (POLY) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = rescale * (cc * w[e] + cb * ((float)gh[q][e] + (float)gl[q][e]));
    }
    half8_t hi, lo;
    split8(w, hi, lo);
    gstore(out + o, hi);
    gstore(out + o + kLo, lo);
    if (i0 != j0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j * Prod::OPITCH + i + e] = w[e];
    }
  }
  if (i0 == j0) return;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PIECES; ++q) {  // the mirror image, four lanes to the 64 bytes of a row's 32 hi (lo)
    const int idx = tid + q * Prod::NT, i = (idx >> 2) % TILE, j = idx / (4 * TILE) * 32 + (idx & 3) * 8;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v[(j + e) * Prod::OPITCH + i];
    half8_t hi, lo;
    split8(w, hi, lo);
    const size_t o = place(i0 + i, j0 + j, a.mp);
    gstore(out + o, hi);
    gstore(out + o + kLo, lo);
  }
}

// x <- a x + P x; the last one writes the result instead
template <int TI, int TJ, int WAVES, typename T, int LAST> __global__ __launch_bounds__(64 * WAVES, 2) void ns_apply_kernel(const Mats* __restrict__ list, int step, float ca, float scale_p, const float* __restrict__ hp) {
  const Mats& t = *list;
  typedef Product<TJ, TI, WAVES, true> Prod;
  __shared__ __attribute__((aligned(16))) char smem[Prod::BYTES];
  const int block = near_tiles(blockIdx.x, gridDim.x), k = find(t, APPLY, block), tid = threadIdx.x, which = step & 1;
  const Mat a = t.mat[k];
  if constexpr (TI == 64 && TJ == 64) {
    if (few(a)) {
      if (step == 0) few_apply<T>(t, a, block - t.first[APPLY][k], reinterpret_cast<double*>(smem), hp);
      return;
    }
  }
  int ti, tj;
  square_tile(block - t.first[APPLY][k], a.mp / TI, a.np / TJ, ti, tj);
  const int i0 = ti * TI, j0 = tj * TJ;
  const ghalf_t* const x = x_of(a, which);
  Prod p;
  p.lds = reinterpret_cast<half_t*>(smem);
  p.run(x + place(0, j0, a.np), a.np, p_of(a) + place(i0, 0, a.mp), a.mp, a.mp, tid);
  constexpr int PIECES = TI * TJ / 8 / Prod::NT;
  half8_t xh[PIECES], xl[PIECES];
#pragma unroll
  for (int q = 0; q < PIECES; ++q) {
    const int idx = tid + q * Prod::NT;
    const size_t o = place(i0 + idx / (TJ / 8), j0 + idx % (TJ / 8) * 8, a.np);
    xh[q] = gload<half8_t>(x + o);
    xl[q] = gload<half8_t>(x + o + kLo);
  }
  float* const v = p.spill(tid);  // v[i][j]
  ghalf_t* const next = x_of(a, which ^ 1);
  const float unscale = 1.f / scale_p;
#pragma unroll
  for (int q = 0; q < PIECES; ++q) {
    const int idx = tid + q * Prod::NT, i = idx / (TJ / 8), j = idx % (TJ / 8) * 8;
    const size_t o = place(i0 + i, j0 + j, a.np);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = fmaf(ca, (float)xh[q][e] + (float)xl[q][e], v[i * Prod::OPITCH + j + e] * unscale);
    if (LAST == 0) {
      half8_t hi, lo;
      split8(w, hi, lo);
      gstore(next + o, hi);
      gstore(next + o + kLo, lo);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i * Prod::OPITCH + j + e] = w[e] * (1.f / kScale);
    }
  }
  if (LAST == 0) return;
  __syncthreads();
  const bool flip = a.rows > a.cols;
  const float lr = LAST == 2 ? hp[2 * a.group] : 0.f, keep = LAST == 2 ? 1.f - lr * hp[2 * a.group + 1] : 0.f, rate = lr * a.gain;
  const int across = flip ? TI : TJ;
  constexpr int IN_FLIGHT = 8;
  for (int base = tid; base < TI * TJ; base += Prod::NT * IN_FLIGHT) {
    float old[IN_FLIGHT];
    size_t o[IN_FLIGHT];
    bool in[IN_FLIGHT];
#pragma unroll
    for (int q = 0; q < IN_FLIGHT; ++q) {
      const int idx = base + q * Prod::NT, slow = idx / across, fast = idx % across, i = flip ? fast : slow, j = flip ? slow : fast;
      in[q] = i0 + i < a.m && j0 + j < a.n;
      o[q] = in[q] ? (flip ? (size_t)(j0 + j) * a.cols + i0 + i : (size_t)(i0 + i) * a.cols + j0 + j) : 0;
      if (LAST == 2) old[q] = gvalue<float>(a.par, o[q]);
    }
#pragma unroll
    for (int q = 0; q < IN_FLIGHT; ++q) {
      const int idx = base + q * Prod::NT, slow = idx / across, fast = idx % across;
      const float y = flip ? v[fast * Prod::OPITCH + slow] : v[slow * Prod::OPITCH + fast];
      if (!in[q]) continue;
      if (LAST == 1) gput<T>(a.dst, o[q], y);
      else gput<float>(a.par, o[q], old[q] * keep - rate * y);
    }
  }
}

int round_up(int v, int to) { return (v + to - 1) / to * to; }
// sides are padded to 64, or to 128 where that adds little: both tile widths then fit
int pad_of(int v) { return v >= 512 ? round_up(v, 128) : round_up(v, 64); }
long long bytes_of(const cvh_ns_matrix& a) {
  const long long m = a.rows < a.cols ? a.rows : a.cols, n = a.rows < a.cols ? a.cols : a.rows;
  const long long mp = pad_of((int)m), np = pad_of((int)n), chunks = (m * n + kNormItems - 1) / kNormItems;
  return (4 * mp * np + 4 * mp * mp) * 2 + (chunks * 8 + 255) / 256 * 256;
}

constexpr long long kListBytes = (sizeof(Mats) + 255) / 256 * 256;
template <typename F> int prefix(Mats& t, int phase, F&& groups) {
  int n = 0;
  for (int i = 0; i <= kMats; ++i) {
    t.first[phase][i] = i <= t.count ? n : 0x7fffffff;
    if (i < t.count) n += groups(t.mat[i]);
  }
  return n;
}
// 128-wide tiles of the symmetric products where there is one for half of the card's 256 units; fewer of them leave more of it idle than the smaller
// tiles cost (all five steps of one matrix, 64- / 128-wide: 1792 x 1792, 105 tiles: 589 / 650 us; 2048 x 2048, 136 tiles: 818 / 754 us).
constexpr int kWideSym = 128;
// P x: 128 x 128 where they come in one round of half of the card or more (1536 x 1536, 144 tiles: 463 us, with 128 x 64 tiles 499, with 64 x 64 486).
// Below and above that 128 x 64, two workgroups a unit: twice as many of them (1280 x 1280, 100 tiles: 287, 322, 302 us), and in several rounds one's
// loads and epilogue under the other's MFMAs (a text tower's 24 matrices, 1152 tiles: 837, 872, 883 us).  64 x 64 below 72 (1024 x 1024, 64 tiles:
// 207 us, with 128 x 64 tiles 230).
enum { SQUARE_64, TALL, SQUARE_128 };
constexpr int kTallLeast = 72, kSquareLeast = 128, kSquareMost = 256;
template <typename F> long long wide_tiles(const Mats& t, F&& tiles) {  // 0: not every side takes them
  long long n = 0;
  for (int i = 0; i < t.count; ++i) {
    if (t.mat[i].mp % 128 || t.mat[i].np % 128) return 0;
    n += tiles(t.mat[i]);
  }
  return n;
}
template <int TILE> int sym_tiles(const Mat& q) { return few(q) ? 1 : q.mp / TILE * (q.mp / TILE + 1) / 2; }
template <int TI, int TJ> int all_tiles(const Mat& q) { return few(q) ? (q.n + kFewCols - 1) / kFewCols : q.mp / TI * (q.np / TJ); }
int scale_tiles(const Mat& q) { return few(q) ? few_chunks(q) : all_tiles<64, 64>(q); }

// What a step's G and P can reach: the singular values in front of it lie in 0 .. most (1 in front of the first step), those behind it in 0 .. the largest
// |a s + b s^3 + c s^5| there.  Each is stored times 2^12 (2^10), or times the largest smaller power of two that keeps it under fp16's 65504 (a tenth of
// it left for rounding): G is the SQUARE of x, 225 where a singular value is 15, and P of the last step whatever the coefficients make of that.  With
// NS_COEFFICIENTS singular values stay below 1.3, and both scales are the large ones.
constexpr double kMostSingular = 15.0;
struct Bounds {
  double a, b, c, most = 1.0;
  Bounds(double a_, double b_, double c_) : a(a_), b(b_), c(c_) {}
  static float scale(double value, float largest) {
    float s = largest;
    while (value * s > 60000.0) s *= 0.5f;
    return s;
  }
  float scale_g() const { return scale(most * most, 4096.f); }
  float scale_p() const {  // of b t + c t^2 for t = s^2: at the end, or at the vertex in front of it
    const double end = most * most, vertex = c != 0.0 ? -b / (2.0 * c) : -1.0;
    return scale(fmax(fabs(b * end + c * end * end), vertex > 0.0 && vertex < end ? fabs(b * vertex / 2.0) : 0.0), 1024.f);
  }
  void step() {
    const double end = most * most;
    double m = fabs(a + b * end + c * end * end) * most;
    auto at = [&](double t) {  // a place where the derivative a + 3 b t + 5 c t^2 is zero
      if (t > 0.0 && t < end) m = fmax(m, fabs(a + b * t + c * t * t) * sqrt(t));
    };
    const double root = 9.0 * b * b - 20.0 * a * c;
    if (c == 0.0) {
      if (b != 0.0) at(-a / (3.0 * b));
    } else if (root >= 0.0) {
      const double q = -0.5 * (3.0 * b + (b < 0.0 ? -sqrt(root) : sqrt(root)));
      at(q / (5.0 * c));
      if (q != 0.0) at(a / q);
    }
    most = m;
  }
};
// singular values stay below kMostSingular in front of every step (behind the last one they may be anything: the result is not an fp16 pair)
bool stays_small(int steps, double a, double b, double c) {
  Bounds bounds(a, b, c);
  for (int s = 1; s < steps; ++s) {
    const double before = bounds.most;
    bounds.step();
    if (!(bounds.most <= kMostSingular)) return false;
    if (bounds.most == before) break;  // the same interval again, for good
  }
  return true;
}

template <int TILE, int WAVES> void run_sym(const Mats* list, int n, int step, bool poly, float b, float c, const Bounds& at, hipStream_t st) {
  ns_sym_kernel<TILE, WAVES, false><<<dim3(n), dim3(64 * WAVES), 0, st>>>(list, step, b, c, at.scale_g(), at.scale_p());
  if (poly) ns_sym_kernel<TILE, WAVES, true><<<dim3(n), dim3(64 * WAVES), 0, st>>>(list, step, b, c, at.scale_g(), at.scale_p());
}
template <typename T, int LAST> void run_apply(int tile, const Mats* list, int n, int step, float a, float scale_p, const float* hp, hipStream_t st) {
  if (tile == SQUARE_128) ns_apply_kernel<128, 128, 8, T, LAST><<<dim3(n), dim3(512), 0, st>>>(list, step, a, scale_p, hp);
  else if (tile == TALL) ns_apply_kernel<128, 64, 4, T, LAST><<<dim3(n), dim3(256), 0, st>>>(list, step, a, scale_p, hp);
  else ns_apply_kernel<64, 64, 4, T, LAST><<<dim3(n), dim3(256), 0, st>>>(list, step, a, scale_p, hp);
}
template <typename T, bool MOM> int run_list(Mats& t, Mats* list, int steps, float a, float b, float c, float eps, float mu, int nesterov, const float* hp, hipStream_t st) {
  const bool ws = wide_tiles(t, sym_tiles<128>) >= kWideSym;
  const long long wide = wide_tiles(t, all_tiles<128, 128>);
  const int wa = wide < kTallLeast ? SQUARE_64 : wide < kSquareLeast || wide > kSquareMost ? TALL : SQUARE_128;
  const int norms = prefix(t, NORM, [](const Mat& q) { return (int)(((long long)q.m * q.n + kNormItems - 1) / kNormItems); });
  const int scales = prefix(t, SCALE, scale_tiles);
  const int syms = ws ? prefix(t, SYM, sym_tiles<128>) : prefix(t, SYM, sym_tiles<64>);
  const int applies = wa == SQUARE_128 ? prefix(t, APPLY, all_tiles<128, 128>) : wa == TALL ? prefix(t, APPLY, all_tiles<128, 64>) : prefix(t, APPLY, all_tiles<64, 64>);
  bool all_few = true;
  for (int i = 0; i < t.count; ++i) all_few = all_few && few(t.mat[i]);
  t.steps = steps; t.nesterov = nesterov; t.a = a; t.b = b; t.c = c; t.eps = eps; t.mu = mu;
  ns_norm_kernel<T, MOM><<<dim3(norms), dim3(256), 0, st>>>(t, list, mu, nesterov);
  ns_scale_kernel<T, MOM><<<dim3(scales), dim3(256), 0, st>>>(list, mu, nesterov, eps);
  constexpr int LAST = MOM ? 2 : 1;
  Bounds at(a, b, c);
  for (int s = 0; s < (all_few ? 1 : steps); ++s, at.step()) {
    if (ws) run_sym<128, 8>(list, syms, s, !all_few, b, c, at, st);
    else run_sym<64, 4>(list, syms, s, !all_few, b, c, at, st);
    if (s + 1 < steps) run_apply<T, 0>(wa, list, applies, s, a, at.scale_p(), hp, st);
    else run_apply<T, LAST>(wa, list, applies, s, a, at.scale_p(), hp, st);
  }
  CVH_CHECK_LAUNCH();
  return 0;
}

template <typename T, bool MOM>
int run_all(const cvh_ns_matrix* mats, int n, int steps, float a, float b, float c, float eps, float mu, int nesterov, const float* hp, void* ws, hipStream_t st) {
  char* at = reinterpret_cast<char*>(ws);
  for (int i0 = 0; i0 < n; i0 += kMats) {
    Mats t = {};
    Mats* const list = reinterpret_cast<Mats*>(at);
    at += kListBytes;
    t.count = n - i0 < kMats ? n - i0 : kMats;
    for (int i = 0; i < t.count; ++i) {
      const cvh_ns_matrix& q = mats[i0 + i];
      Mat& d = t.mat[i];
      d.src = q.src; d.dst = q.dst; d.mom = q.momentum; d.par = q.param;
      d.rows = q.rows; d.cols = q.cols; d.group = q.group; d.gain = q.gain;
      d.m = q.rows < q.cols ? q.rows : q.cols;
      d.n = q.rows < q.cols ? q.cols : q.rows;
      d.mp = pad_of(d.m);
      d.np = pad_of(d.n);
      d.ws = reinterpret_cast<half_t*>(at);
      d.norm = reinterpret_cast<double*>(at + (4ll * d.mp * d.np + 4ll * d.mp * d.mp) * 2);
      at += bytes_of(q);
    }
    const int rc = run_list<T, MOM>(t, list, steps, a, b, c, eps, mu, nesterov, hp, st);
    if (rc) return rc;
  }
  return 0;
}

int check(const cvh_ns_matrix* mats, int n, int steps, float a, float b, float c, float eps, bool step) {
  if (mats == nullptr || n <= 0 || steps <= 0 || !(eps >= 0.f) || !(fabsf(a) + fabsf(b) + fabsf(c) <= 15.f) || !stays_small(steps, a, b, c)) return -2;
  for (int i = 0; i < n; ++i) {
    const cvh_ns_matrix& q = mats[i];
    if (q.rows <= 0 || q.cols <= 0 || (q.rows > kMostRows && q.cols > kMostRows) || q.rows > kMostCols || q.cols > kMostCols || q.src == nullptr) return -2;
    if (step ? (q.momentum == nullptr || q.param == nullptr || q.group < 0) : q.dst == nullptr) return -2;
  }
  return 0;
}

}  // namespace

extern "C" int cvh_ns_bounded(int steps, float a, float b, float c) { return steps > 0 && stays_small(steps, a, b, c) ? 1 : 0; }
extern "C" long long cvh_ns_workspace_elems(const cvh_ns_matrix* mats, int n) {
  if (mats == nullptr || n <= 0) return -2;
  long long bytes = (n + kMats - 1) / kMats * kListBytes;
  for (int i = 0; i < n; ++i) bytes += bytes_of(mats[i]);
  return (bytes + 3) / 4;
}
extern "C" int cvh_orthogonalize(int dtype, const cvh_ns_matrix* mats, int n, int steps, float a, float b, float c, float eps, float* ws, void* stream) {
  if (dtype != CVH_DT_F32 && dtype != CVH_DT_BF16) return -1;
  if (int rc = check(mats, n, steps, a, b, c, eps, false)) return rc;
  if (ws == nullptr) return -2;
  return dtype == CVH_DT_BF16 ? run_all<bf16_t, false>(mats, n, steps, a, b, c, eps, 0.f, 0, nullptr, ws, (hipStream_t)stream)
                              : run_all<float, false>(mats, n, steps, a, b, c, eps, 0.f, 0, nullptr, ws, (hipStream_t)stream);
}
extern "C" int cvh_muon_step(const cvh_ns_matrix* mats, int n, int steps, float a, float b, float c, float eps, float momentum, int nesterov, const float* group_hp,
                             float* ws, void* stream) {
  if (int rc = check(mats, n, steps, a, b, c, eps, true)) return rc;
  if (ws == nullptr || group_hp == nullptr || !(momentum >= 0.f && momentum < 1.f)) return -2;
  return run_all<float, true>(mats, n, steps, a, b, c, eps, momentum, nesterov, group_hp, ws, (hipStream_t)stream);
}
