// Orthogonalised updates: Newton-Schulz products on a list of matrices, and the optimizer step around them.
//
//   u = g  (orthogonalize)   or   mom <- mu mom + g,  u = g + mu mom (Nesterov) or mom  (optimizer step)
//   x <- u / (|u|_F + eps), the shorter side m as rows;   `steps` times:  G = x x^T,  P = b G + c G G,  x <- a x + P x
//   result = x   or   w <- (1 - lr wd) w - lr gain x
//
// G and P are symmetric and commute: half of their tiles are computed and written twice.  Operands are kept as pairs of fp16 numbers, hi + lo,
// of the value times a power of two (2^12 for x and G, 2^10 for P: singular values below 16 and |P|_2 below 64 stay under fp16's 65504, and an
// entry of ordinary size stays far above its subnormals): 22 bits and a sign, and a product is three MFMAs, hi hi + hi lo + lo hi, accumulated in float32 - within a factor of two of a
// float32 product's error, at a third of the fp16 matrix rate instead of the float32 matrix rate (measured on 8192-cubed library products: 1081 / 3
// = 360 against 154 TFLOP/s).  One fp16 or bf16 product per step would be three times as fast, and its rounding (2^-11 and 2^-8) is multiplied by up to
// a^steps = 485 in the directions of small singular values.
//
// (a x is added to the finished sum: with a I inside P the small terms of the long sum are rounded next to a x, 8e-6 instead of 2e-6 after 5
// steps of a 1030 x 1100 matrix, whose float32 products give 2e-6, too.)
// x is kept in both layouts, [m][n] and [n][m], so that every product is rows times rows with the contraction index contiguous; the epilogue
// writes both.  Sides are padded to the tile with zeros, which the products keep zero, so that the main loop has no bounds.
// All matrices of a list go through one launch per product (a table in the kernel's arguments): 2 + 3 steps launches for up to kMats matrices.
#include "common.hpp"
#include "cvnets_hip.h"

namespace {

constexpr int kMats = 32;
constexpr int kMostRows = 1 << 14, kMostCols = 1 << 24;  // of the shorter and the longer side
constexpr float kScale = 4096.f, kScaleP = 1024.f;  // of x and G; of P
typedef _Float16 half_t;
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

struct Mat {
  const void* src;  // u, or the gradient (float32)
  void* dst;        // result (orthogonalize)
  float *mom, *par;
  half_t* ws;       // x [2][mp][np], x^T [2][np][mp], the same again (ping-pong), G [2][mp][mp], P [2][mp][mp]; hi and lo planes
  double* norm;     // partial sums of squares
  int m, n, mp, np, rows, cols, group;
  float gain;
};
struct Mats {
  Mat mat[kMats];
  int first[kMats + 1];  // prefix of workgroups
  int count;
};
__device__ __forceinline__ int find(const Mats& t, int wg) {
  int i = 0;
  while (i + 1 < t.count && wg >= t.first[i + 1]) ++i;
  return i;
}
__device__ __forceinline__ size_t plane_x(const Mat& a) { return (size_t)a.mp * a.np; }
__device__ __forceinline__ half_t* x_of(const Mat& a, int which) { return a.ws + (size_t)which * 4 * plane_x(a); }
__device__ __forceinline__ half_t* xt_of(const Mat& a, int which) { return x_of(a, which) + 2 * plane_x(a); }
__device__ __forceinline__ half_t* g_of(const Mat& a) { return a.ws + 8 * plane_x(a); }
__device__ __forceinline__ half_t* p_of(const Mat& a) { return g_of(a) + 2 * (size_t)a.mp * a.mp; }

__device__ __forceinline__ void split(float v, half_t& hi, half_t& lo) {
  hi = (half_t)v;
  lo = (half_t)(v - (float)hi);
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// sums of squares (and the momentum), kNormItems elements a workgroup; in 64 bits, so that no gradient's square leaves the range
// -----------------------------------------------------------------------------------------------------------------------------------------
constexpr int kNormItems = 16384;
template <typename T, bool MOM> __device__ __forceinline__ float update_of(const Mat& a, size_t i, float mu, int nesterov) {
  const float g = to_f<T>(reinterpret_cast<const T*>(a.src)[i]);
  if (!MOM) return g;
  const float m = a.mom[i];
  return nesterov ? g + mu * m : m;
}
template <typename T, bool MOM> __global__ __launch_bounds__(256) void ns_norm_kernel(Mats t, float mu, int nesterov) {
  __shared__ double sums[4];
  const int k = find(t, blockIdx.x), chunk = blockIdx.x - t.first[k];
  const Mat& a = t.mat[k];
  const size_t size = (size_t)a.m * a.n, i0 = (size_t)chunk * kNormItems, i1 = i0 + kNormItems < size ? i0 + kNormItems : size;
  double s = 0.0;
  for (size_t i = i0 + threadIdx.x; i < i1; i += 256) {
    if (MOM) a.mom[i] = mu * a.mom[i] + to_f<T>(reinterpret_cast<const T*>(a.src)[i]);
    const double u = update_of<T, MOM>(a, i, mu, nesterov);
    s += u * u;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.norm[chunk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// x = u / (|u| + eps) into both layouts, 64 x 64 elements (of the padded matrix) a workgroup
// -----------------------------------------------------------------------------------------------------------------------------------------
template <typename T, bool MOM> __global__ __launch_bounds__(256) void ns_scale_kernel(Mats t, float mu, int nesterov, float eps) {
  __shared__ float tile[64][65];
  __shared__ double total;
  const int k = find(t, blockIdx.x), at = blockIdx.x - t.first[k], tid = threadIdx.x;
  const Mat& a = t.mat[k];
  const int tn = a.np / 64, i0 = at / tn * 64, j0 = at % tn * 64;
  if (tid < 64) {
    const int chunks = (int)(((size_t)a.m * a.n + kNormItems - 1) / kNormItems);
    double s = 0.0;
    for (int c = tid; c < chunks; c += 64) s += a.norm[c];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (tid == 0) total = s;
  }
  const bool flip = a.rows > a.cols;  // x[i][j] = u[j][i]
  for (int e = tid; e < 4096; e += 256) {
    const int r = e >> 6, c = e & 63;  // of u's tile: c runs along u's rows
    const int i = flip ? i0 + c : i0 + r, j = flip ? j0 + r : j0 + c;
    const float v = i < a.m && j < a.n ? update_of<T, MOM>(a, (size_t)(flip ? j : i) * a.cols + (flip ? i : j), mu, nesterov) : 0.f;
    if (flip) tile[c][r] = v; else tile[r][c] = v;
  }
  __syncthreads();
  const double inv = (double)kScale / (sqrt(total) + (double)eps);
  half_t *x = x_of(a, 0), *xt = xt_of(a, 0);
  const size_t plane = plane_x(a);
  for (int e = tid; e < 4096; e += 256) {
    const int r = e >> 6, c = e & 63;
    half_t hi, lo;
    split((float)(tile[r][c] * inv), hi, lo);
    const size_t o = (size_t)(i0 + r) * a.np + j0 + c;
    x[o] = hi;
    x[plane + o] = lo;
    split((float)(tile[c][r] * inv), hi, lo);
    const size_t p = (size_t)(j0 + r) * a.mp + i0 + c;
    xt[p] = hi;
    xt[plane + p] = lo;
  }
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// rows-times-rows product of hi + lo operands: acc[i][j] = sum_k A[i][k] B[j][k] for a TILE x TILE tile, 4 waves of (TILE / 2)^2
// -----------------------------------------------------------------------------------------------------------------------------------------
constexpr int BK = 32, PITCH = BK + 8;
template <int TILE> struct Product {
  static constexpr int W = TILE / 64;       // 32-wide fragments of a wave in each direction
  static constexpr int CH = TILE * (BK / 8) / 256;  // 16-byte pieces a thread loads of each plane
  half_t* lds;                              // [2 stages][4 planes: A hi, A lo, B hi, B lo][TILE][PITCH]
  f32x16_t acc[W][W];
  uint4 q[4][CH];

  __device__ __forceinline__ void load(const half_t* a, size_t a_plane, int lda, const half_t* b, size_t b_plane, int ldb, int k0, int tid) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int idx = tid + c * 256, r = idx >> 2, col = k0 + (idx & 3) * 8;
      q[0][c] = *reinterpret_cast<const uint4*>(a + (size_t)r * lda + col);
      q[1][c] = *reinterpret_cast<const uint4*>(a + a_plane + (size_t)r * lda + col);
      q[2][c] = *reinterpret_cast<const uint4*>(b + (size_t)r * ldb + col);
      q[3][c] = *reinterpret_cast<const uint4*>(b + b_plane + (size_t)r * ldb + col);
    }
  }
  __device__ __forceinline__ void store(int stage, int tid) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int idx = tid + c * 256;
        *reinterpret_cast<uint4*>(lds + ((size_t)(stage * 4 + p) * TILE + (idx >> 2)) * PITCH + (idx & 3) * 8) = q[p][c];
      }
  }
  __device__ __forceinline__ half8_t frag(int stage, int plane, int row, int k, int lane) const {
    return *reinterpret_cast<const half8_t*>(lds + ((size_t)(stage * 4 + plane) * TILE + row + (lane & 31)) * PITCH + k + 8 * (lane >> 5));
  }
  __device__ __forceinline__ void run(const half_t* a, size_t a_plane, int lda, const half_t* b, size_t b_plane, int ldb, int K, int tid) {
    const int lane = tid & 63, wr = (tid >> 7) * (TILE / 2), wc = ((tid >> 6) & 1) * (TILE / 2);
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) acc[i][j] = acc_zero();
    load(a, a_plane, lda, b, b_plane, ldb, 0, tid);
    store(0, tid);
    if (K > BK) load(a, a_plane, lda, b, b_plane, ldb, BK, tid);
    for (int k0 = 0, s = 0; k0 < K; k0 += BK, s ^= 1) {
      wg_barrier_lds();
      if (k0 + BK < K) store(s ^ 1, tid);
      if (k0 + 2 * BK < K) load(a, a_plane, lda, b, b_plane, ldb, k0 + 2 * BK, tid);
#pragma unroll
      for (int k = 0; k < BK; k += 16) {
        half8_t ah[W], al[W], bh[W], bl[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
          ah[i] = frag(s, 0, wr + 32 * i, k, lane);
          al[i] = frag(s, 1, wr + 32 * i, k, lane);
          bh[i] = frag(s, 2, wc + 32 * i, k, lane);
          bl[i] = frag(s, 3, wc + 32 * i, k, lane);
        }
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
          for (int j = 0; j < W; ++j) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
          }
      }
    }
  }
  // f(row, column, 4 values of rows row .. row + 3) over the tile
  template <typename F> __device__ __forceinline__ void each(int tid, F&& f) const {
    const int lane = tid & 63, wr = (tid >> 7) * (TILE / 2), wc = ((tid >> 6) & 1) * (TILE / 2);
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const float v[4] = {acc[i][j][4 * q4], acc[i][j][4 * q4 + 1], acc[i][j][4 * q4 + 2], acc[i][j][4 * q4 + 3]};
          f(wr + 32 * i + 8 * q4 + 4 * (lane >> 5), wc + 32 * j + (lane & 31), v);
        }
  }
};

// value[i .. i + 3][j] as hi + lo into both an [i][j] and a [j][i] matrix
__device__ __forceinline__ void put(half_t* ij, size_t ij_plane, int ld_ij, half_t* ji, size_t ji_plane, int ld_ji, int i, int j, const float* v) {
  half4_t hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    half_t h, l;
    split(v[e], h, l);
    hi[e] = h;
    lo[e] = l;
    if (ij != nullptr) {
      ij[(size_t)(i + e) * ld_ij + j] = h;
      ij[ij_plane + (size_t)(i + e) * ld_ij + j] = l;
    }
  }
  if (ji != nullptr) {
    *reinterpret_cast<half4_t*>(ji + (size_t)j * ld_ji + i) = hi;
    *reinterpret_cast<half4_t*>(ji + ji_plane + (size_t)j * ld_ji + i) = lo;
  }
}

// G = x x^T (POLY false) or P = b G + c G G (true): tiles (i, j <= i), written to both halves
template <int TILE, bool POLY> __global__ __launch_bounds__(256, 2) void ns_sym_kernel(Mats t, int which, float cb, float cc) {
  __shared__ __attribute__((aligned(16))) half_t lds[2 * 4 * TILE * PITCH];
  const int k = find(t, blockIdx.x), tid = threadIdx.x;
  const Mat& a = t.mat[k];
  int at = blockIdx.x - t.first[k], ti = 0;
  while (at > ti) at -= ++ti;  // (ti, at) of the lower triangle
  const int i0 = ti * TILE, j0 = at * TILE;
  const size_t plane = (size_t)a.mp * a.mp;
  half_t* const g = g_of(a);
  Product<TILE> p;
  p.lds = lds;
  if (POLY) p.run(g + (size_t)i0 * a.mp, plane, a.mp, g + (size_t)j0 * a.mp, plane, a.mp, a.mp, tid);
  else p.run(x_of(a, which) + (size_t)i0 * a.np, plane_x(a), a.np, x_of(a, which) + (size_t)j0 * a.np, plane_x(a), a.np, a.np, tid);
  half_t* const out = POLY ? p_of(a) : g;
  p.each(tid, [&](int i, int j, const float* v) {
    float w[4];
    if (POLY) {
      const size_t o = (size_t)(j0 + j) * a.mp + i0 + i;  // G[j][i ..] = G[i ..][j]
      const half4_t h = *reinterpret_cast<const half4_t*>(g + o), l = *reinterpret_cast<const half4_t*>(g + plane + o);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = (kScaleP / kScale) * (cc * (v[e] * (1.f / kScale)) + cb * ((float)h[e] + (float)l[e]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = v[e] * (1.f / kScale);
    }
    put(i0 == j0 ? nullptr : out, plane, a.mp, out, plane, a.mp, i0 + i, j0 + j, w);
  });
}

// x <- a x + P x; the last one writes the result instead
template <int TILE, typename T, int LAST> __global__ __launch_bounds__(256, 2) void ns_apply_kernel(Mats t, int which, float ca, const float* __restrict__ hp) {
  __shared__ __attribute__((aligned(16))) half_t lds[2 * 4 * TILE * PITCH];
  const int k = find(t, blockIdx.x), tid = threadIdx.x, at = blockIdx.x - t.first[k];
  const Mat& a = t.mat[k];
  const int tm = a.mp / TILE, i0 = at % tm * TILE, j0 = at / tm * TILE;
  Product<TILE> p;
  p.lds = lds;
  p.run(p_of(a) + (size_t)i0 * a.mp, (size_t)a.mp * a.mp, a.mp, xt_of(a, which) + (size_t)j0 * a.mp, plane_x(a), a.mp, a.mp, tid);
  const half_t* const xt = xt_of(a, which);
  const size_t plane = plane_x(a);
  auto next = [&](int i, int j, const float* v, float* w) {  // kScale times the new x[i .. i + 3][j]
    const size_t o = (size_t)(j0 + j) * a.mp + i0 + i;
    const half4_t h = *reinterpret_cast<const half4_t*>(xt + o), l = *reinterpret_cast<const half4_t*>(xt + plane + o);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = fmaf(ca, (float)h[e] + (float)l[e], v[e] * (1.f / kScaleP));
  };
  if (LAST == 0) {
    p.each(tid, [&](int i, int j, const float* v) {
      float w[4];
      next(i, j, v, w);
      put(x_of(a, which ^ 1), plane_x(a), a.np, xt_of(a, which ^ 1), plane_x(a), a.mp, i0 + i, j0 + j, w);
    });
  } else {
    const bool flip = a.rows > a.cols;
    const float lr = LAST == 2 ? hp[2 * a.group] : 0.f, keep = LAST == 2 ? 1.f - lr * hp[2 * a.group + 1] : 0.f, step = lr * a.gain;
    p.each(tid, [&](int i, int j, const float* v) {
      float w[4];
      next(i, j, v, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = i0 + i + e, c = j0 + j;
        if (r >= a.m || c >= a.n) continue;
        const size_t o = flip ? (size_t)c * a.cols + r : (size_t)r * a.cols + c;
        const float x = w[e] * (1.f / kScale);
        if (LAST == 1) reinterpret_cast<T*>(a.dst)[o] = from_f<T>(x);
        else a.par[o] = a.par[o] * keep - step * x;
      }
    });
  }
}

int round_up(int v, int to) { return (v + to - 1) / to * to; }
// 128-wide tiles unless the list has too few of them for the card; then 64-wide ones (and no side is padded to more than it has to be)
int tile_of(const cvh_ns_matrix* mats, int n) {
  long long tiles = 0;
  for (int i = 0; i < n; ++i) {
    const int m = mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols, w = mats[i].rows < mats[i].cols ? mats[i].cols : mats[i].rows;
    tiles += (long long)(round_up(m, 128) / 128) * (round_up(w, 128) / 128);
  }
  return tiles >= 512 ? 128 : 64;
}
long long bytes_of(const cvh_ns_matrix& a, int tile) {
  const long long m = a.rows < a.cols ? a.rows : a.cols, n = a.rows < a.cols ? a.cols : a.rows;
  const long long mp = round_up((int)m, tile), np = round_up((int)n, tile), chunks = (m * n + kNormItems - 1) / kNormItems;
  return (8 * mp * np + 4 * mp * mp) * 2 + (chunks * 8 + 255) / 256 * 256;
}

template <typename F> void prefix(Mats& t, F&& groups) {
  t.first[0] = 0;
  for (int i = 0; i < t.count; ++i) t.first[i + 1] = t.first[i] + groups(t.mat[i]);
}
template <int TILE, typename T, bool MOM> int run_list(Mats& t, int steps, float a, float b, float c, float eps, float mu, int nesterov, const float* hp, hipStream_t st) {
  prefix(t, [](const Mat& q) { return (int)(((long long)q.m * q.n + kNormItems - 1) / kNormItems); });
  ns_norm_kernel<T, MOM><<<dim3(t.first[t.count]), dim3(256), 0, st>>>(t, mu, nesterov);
  prefix(t, [](const Mat& q) { return q.mp / 64 * (q.np / 64); });
  ns_scale_kernel<T, MOM><<<dim3(t.first[t.count]), dim3(256), 0, st>>>(t, mu, nesterov, eps);
  Mats sym = t;
  prefix(sym, [](const Mat& q) { return q.mp / TILE * (q.mp / TILE + 1) / 2; });
  prefix(t, [](const Mat& q) { return q.mp / TILE * (q.np / TILE); });
  const dim3 gs(sym.first[sym.count]), ga(t.first[t.count]);
  for (int s = 0; s < steps; ++s) {
    ns_sym_kernel<TILE, false><<<gs, dim3(256), 0, st>>>(sym, s & 1, b, c);
    ns_sym_kernel<TILE, true><<<gs, dim3(256), 0, st>>>(sym, s & 1, b, c);
    if (s + 1 < steps) ns_apply_kernel<TILE, T, 0><<<ga, dim3(256), 0, st>>>(t, s & 1, a, hp);
    else ns_apply_kernel<TILE, T, MOM ? 2 : 1><<<ga, dim3(256), 0, st>>>(t, s & 1, a, hp);
  }
  CVH_CHECK_LAUNCH();
  return 0;
}

template <typename T, bool MOM>
int run_all(const cvh_ns_matrix* mats, int n, int steps, float a, float b, float c, float eps, float mu, int nesterov, const float* hp, void* ws, hipStream_t st) {
  const int tile = tile_of(mats, n);
  char* at = reinterpret_cast<char*>(ws);
  for (int i0 = 0; i0 < n; i0 += kMats) {
    Mats t;
    t.count = n - i0 < kMats ? n - i0 : kMats;
    for (int i = 0; i < t.count; ++i) {
      const cvh_ns_matrix& q = mats[i0 + i];
      Mat& d = t.mat[i];
      d.src = q.src; d.dst = q.dst; d.mom = q.momentum; d.par = q.param;
      d.rows = q.rows; d.cols = q.cols; d.group = q.group; d.gain = q.gain;
      d.m = q.rows < q.cols ? q.rows : q.cols;
      d.n = q.rows < q.cols ? q.cols : q.rows;
      d.mp = round_up(d.m, tile);
      d.np = round_up(d.n, tile);
      d.ws = reinterpret_cast<half_t*>(at);
      d.norm = reinterpret_cast<double*>(at + (8ll * d.mp * d.np + 4ll * d.mp * d.mp) * 2);
      at += bytes_of(q, tile);
    }
    const int rc = tile == 128 ? run_list<128, T, MOM>(t, steps, a, b, c, eps, mu, nesterov, hp, st) : run_list<64, T, MOM>(t, steps, a, b, c, eps, mu, nesterov, hp, st);
    if (rc) return rc;
  }
  return 0;
}

int check(const cvh_ns_matrix* mats, int n, int steps, float a, float b, float c, float eps, bool step) {
  if (mats == nullptr || n <= 0 || steps <= 0 || !(eps >= 0.f) || !(fabsf(a) + fabsf(b) + fabsf(c) <= 15.f)) return -2;
  for (int i = 0; i < n; ++i) {
    const cvh_ns_matrix& q = mats[i];
    if (q.rows <= 0 || q.cols <= 0 || (q.rows > kMostRows && q.cols > kMostRows) || q.rows > kMostCols || q.cols > kMostCols || q.src == nullptr) return -2;
    if (step ? (q.momentum == nullptr || q.param == nullptr || q.group < 0) : q.dst == nullptr) return -2;
  }
  return 0;
}

}  // namespace

extern "C" long long cvh_ns_workspace_elems(const cvh_ns_matrix* mats, int n) {
  if (mats == nullptr || n <= 0) return -2;
  long long bytes = 0;
  const int tile = tile_of(mats, n);
  for (int i = 0; i < n; ++i) bytes += bytes_of(mats[i], tile);
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
