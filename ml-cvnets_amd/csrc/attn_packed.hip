// Softmax attention over PACKED sequences of different lengths (grouped query heads, causal or not), forward + backward, on MFMA.
//
//   s_ij = scale q_i . k_j  (j in i's sequence, j <= i when causal)    p = softmax_j(s)    o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i     ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i     dq_i = scale sum_j ds_ij k_j     dk_j = scale sum_i ds_ij q_i
//
// q [rows][hq][d], k / v [rows][hkv][d] (any row / head stride, d contiguous); the sequences lie one behind the other, sequence b in rows
// cu[b] .. cu[b + 1] - 1.  The scores never reach memory: one pass over the keys with a running maximum and sum (forward), and a
// recomputation from the stored log-sum in the two backward kernels.  dk / dv of a key head are summed over its query heads inside ONE
// workgroup (a loop over the group), so nothing is accumulated with atomics and every result is bit-reproducible.
//
// A wave owns 32 queries (forward, dq) or 32 keys (dk / dv) and forms TRANSPOSED products: S^T = K Q^T has the query along lane & 31, so the
// softmax statistics are per-lane scalars, and the accumulator rows of P^T are the contraction index of O^T = V^T P^T: the probabilities go
// from accumulator to operand registers and never touch LDS.  The waves of a workgroup share the staged K / V (or Q / dO) tiles, which are
// double-buffered in LDS and loaded a tile ahead through registers.
//
// What bounds it (measured, MI355X): 128 columns, 20 k rows in 3 documents, 16 / 4 heads, causal forward: 600 .. 640 us (cards differ) = 966 .. 905
// TFLOP/s of the 4 d a pair that have to be computed; MFMA 48 %, arithmetic 43 %, LDS 48 % of the cycles, which two waves a SIMD overlap only in part.  Training
// there: 2800 .. 2930 us.  64 columns, 24.6 k rows, 12 / 4 heads, training: forward 93, dq 134, dk / dv 169 us; a score costs an exponential and three other operations next to 1 / 4 of an MFMA.  128-row
// workgroups: 4 waves share each staged tile; 64 keys (queries) a tile: at 64 columns 32 cost 20 % and 128 10 % in dk / dv, at 96 and 128 columns 32 cost 5 .. 8 % of
// a whole training pass.  Captions (5 .. 77 tokens): one wave per 32 rows, 20 + 27 + 21 us for 13 k rows x 8 heads, latency.
//
// Work items come from a plan (packed_plan_kernel) made once per batch: (sequence, block) pairs, most expensive first, so that the last
// workgroups to start are the short ones; the list also has the rows behind the last sequence, whose results are written as zeros.
#include "common.hpp"
#include "cvnets_hip.h"

namespace {

typedef cvh_packed_attn PA;

__device__ __forceinline__ float pexp2(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kL2E = 1.4426950408889634f;

template <typename T> struct Chunk;  // 16 bytes
template <> struct Chunk<bf16_t> {
  static constexpr int N = 8;
};
template <> struct Chunk<float> {
  static constexpr int N = 4;
};

// Rows of one sequence through a buffer descriptor: what lies at or behind `bytes` reads as zero without an access.  A masked probability is 0, and
// 0 times whatever another sequence holds there has to be 0; and no load of the loops needs a bounds test, a mask or a branch - behind a
// branch the compiler's counts of outstanding loads are lower bounds and it waits for the newest load instead of the oldest.
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr int kBeyond = 0x7ffffff0;  // an offset that no descriptor covers
__device__ __forceinline__ rsrc_t rows_of(const void* base, long long bytes) {
  const long long most = kBeyond;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)(bytes < 0 ? 0 : bytes < most ? bytes : most), 0x00020000);
}
template <typename T> __device__ __forceinline__ rsrc_t tile_rows(const T* seq_base, long long row_stride, int row0, int len, int d) {
  const long long rows = len - row0;
  return rows_of(seq_base + (rows > 0 ? (long long)row0 * row_stride : 0ll), rows > 0 ? ((rows - 1) * row_stride + d) * (long long)sizeof(T) : 0ll);
}
__device__ __forceinline__ uint4 buf16(rsrc_t r, int offset) {
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  const u4 v = __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0);
  return make_uint4(v.x, v.y, v.z, v.w);
}

// one MFMA operand (32 rows x 16 columns) straight from global memory: lane l holds columns k0 + 8 (l >> 5) .. + 7 of row (l & 31); `offset` is the
// byte offset of the lane's row, kBeyond for none
__device__ __forceinline__ Frag<bf16_t> gfrag(rsrc_t r, int offset, int c0, int d, const bf16_t*) {
  Frag<bf16_t> f;
  f.v = __builtin_bit_cast(bf16x8_t, buf16(r, c0 < d ? offset + c0 * 2 : kBeyond));
  return f;
}
__device__ __forceinline__ Frag<float> gfrag(rsrc_t r, int offset, int c0, int d, const float*) {
  Frag<float> f;
  const uint4 a = buf16(r, c0 < d ? offset + c0 * 4 : kBeyond), b = buf16(r, c0 < d ? offset + c0 * 4 + 16 : kBeyond);
  f.v[0] = __uint_as_float(a.x); f.v[1] = __uint_as_float(a.y); f.v[2] = __uint_as_float(a.z); f.v[3] = __uint_as_float(a.w);
  f.v[4] = __uint_as_float(b.x); f.v[5] = __uint_as_float(b.y); f.v[6] = __uint_as_float(b.z); f.v[7] = __uint_as_float(b.w);
  return f;
}
__device__ __forceinline__ float frag_dot(const Frag<bf16_t>& a, const Frag<bf16_t>& b) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += (float)a.v[j] * (float)b.v[j];
  return s;
}
__device__ __forceinline__ float frag_dot(const Frag<float>& a, const Frag<float>& b) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += a.v[j] * b.v[j];
  return s;
}

// LDS tiles of rows x CP columns and their two kinds of operand fragments:
//   rows(row0, k0):  lane l reads columns k0 + 8 (l >> 5) .. + 7 of row row0 + (l & 31)
//   cols(k0, col0):  the TRANSPOSE: column col0 + (l & 31), its rows in the order in which a 32x32 accumulator holds them: slot j of lane half h is row
//                    k0 + 8 (j >> 2) + 4 h + (j & 3).  bf16: two LDS transpose reads (lane 4 r + q of a 16-lane group gives the address of 4 columns of
//                    block row r and receives column 4 r + q of the 4 x 16 block).
// bf16 rows are padded for the row reads, 16 rows x 16 bytes on distinct banks (the pitch an odd number of 16-byte units); the transpose reads, 4 rows x 64
// bytes, would want another pitch (64 bytes past a multiple of 256) and conflict in a quarter of the LDS cycles, which do not bound the kernels.  16 bytes of
// padding for 64 and 96 columns, 48 for 128 (half of the LDS cycles were conflicts with 16).  (An XOR of the 16-byte chunks with the row does the same without padding, at 30
// more registers for the addresses: 164 instead of 128 and spills at 128 columns.)
typedef short v4s_t __attribute__((ext_vector_type(4)));
template <typename T, int CP> struct Tile;
template <int CP> struct Tile<bf16_t, CP> {
  static constexpr int PT = CP == 128 || CP == 32 ? CP + 24 : CP + 8;  // elements a row
  int row_at, col_at;
  static __device__ __forceinline__ int chunk_at(int row, int chunk) { return row * PT + chunk * 8; }
  __device__ __forceinline__ explicit Tile(int lane) {
    const int i = lane & 15;
    row_at = (lane & 31) * PT + 8 * (lane >> 5);
    col_at = (4 * (lane >> 5) + (i >> 2)) * PT + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
  }
  __device__ __forceinline__ Frag<bf16_t> rows(const bf16_t* tile, int row0, int k0) const {
    Frag<bf16_t> r;
    r.v = *reinterpret_cast<const bf16x8_t*>(tile + row_at + row0 * PT + k0);
    return r;
  }
  __device__ __forceinline__ Frag<bf16_t> cols(const bf16_t* tile, int k0, int col0) const {
    const bf16_t* const p = tile + col_at + k0 * PT + col0;
    const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_t*)(p));
    const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_t*)(p + 8 * PT));
    Frag<bf16_t> r;
    r.v = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    return r;
  }
};
template <int CP> struct Tile<float, CP> {
  static constexpr int PT = lds_pitch<float>(CP);
  int lane;
  static __device__ __forceinline__ int chunk_at(int row, int chunk) { return row * PT + chunk * 4; }
  __device__ __forceinline__ explicit Tile(int l) : lane(l) {}
  __device__ __forceinline__ Frag<float> rows(const float* tile, int row0, int k0) const { return lds_frag(tile, PT, row0, k0, lane); }
  __device__ __forceinline__ Frag<float> cols(const float* tile, int k0, int col0) const {
    const float* p = tile + (k0 + 4 * (lane >> 5)) * PT + col0 + (lane & 31);
    Frag<float> r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = p[((j & 3) + 8 * (j >> 2)) * PT];
    return r;
  }
};
// A tile of NROWS consecutive rows of a sequence, loaded by NT threads into registers (load: only issues the reads) and written to LDS (store);
// rows behind the sequence and columns at or behind d are zeros
template <typename T, int CP, int NROWS, int NT> struct RowTile {
  static constexpr int VN = Chunk<T>::N, CH = CP / VN, IT = (NROWS * CH + NT - 1) / NT;
  static constexpr bool EXACT = (NROWS * CH) % NT == 0;
  uint4 q[IT];
  int offset[IT];        // bytes
  const T* base;         // of the tile that is loaded next
  long long left, step;  // bytes of the sequence from there, and of a tile's rows
  __device__ __forceinline__ void start(const T* seq_base, long long row_stride, int row0, int len, int d) {
    base = seq_base + (long long)row0 * row_stride;
    left = ((long long)(len - row0 - 1) * row_stride + d) * (long long)sizeof(T);
    step = NROWS * row_stride * (long long)sizeof(T);
  }
  __device__ __forceinline__ void place(long long row_stride, int d, int tid) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int idx = tid + i * NT, r = idx / CH, c = (idx % CH) * VN;
      offset[i] = (EXACT || idx < NROWS * CH) && c < d ? (r * (int)row_stride + c) * (int)sizeof(T) : kBeyond;
    }
  }
  __device__ __forceinline__ void load() {
    const rsrc_t rows = rows_of(base, left);
#pragma unroll
    for (int i = 0; i < IT; ++i) q[i] = buf16(rows, offset[i]);
    base = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + step);
    left -= step;
  }
  __device__ __forceinline__ void store(T* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int idx = tid + i * NT;
      if (EXACT || idx < NROWS * CH) *reinterpret_cast<uint4*>(lds + Tile<T, CP>::chunk_at(idx / CH, idx % CH)) = q[i];
    }
  }
};

// rows 16 t .. 16 t + 15 (in that order) of an accumulator as an operand.  bf16: the one rounding of P / dS to 8 bits, each probability off by
// at most 2^-8 of itself; the sums it enters stay in 32 bits.
template <typename T> __device__ __forceinline__ Frag<T> acc_frag(const f32x16_t& a, int t);
template <> __device__ __forceinline__ Frag<bf16_t> acc_frag<bf16_t>(const f32x16_t& a, int t) {
  Frag<bf16_t> f;
  f.v = __builtin_bit_cast(bf16x8_t, make_uint4(f2bf_pk(a[8 * t], a[8 * t + 1]), f2bf_pk(a[8 * t + 2], a[8 * t + 3]), f2bf_pk(a[8 * t + 4], a[8 * t + 5]),
                                                f2bf_pk(a[8 * t + 6], a[8 * t + 7])));
  return f;
}
template <> __device__ __forceinline__ Frag<float> acc_frag<float>(const f32x16_t& a, int t) {
  Frag<float> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = a[8 * t + j];
  return f;
}

// the halves of a wave hold 4 + 4 of 8 consecutive columns: lane l and l + 32 exchange, so that each has 8 of one 16-column group
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r.x;
  b = r.y;
}
// f(x of the lane, x of the lane in the other half)
__device__ __forceinline__ float both_halves_max(float x) {
  uint32_t a = __float_as_uint(x), b = a;
  swap_halves(a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float both_halves_sum(float x) {
  uint32_t a = __float_as_uint(x), b = a;
  swap_halves(a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}
// rows of a transposed accumulator: lane = row, registers = 32 columns from c0; `lo` (nullable): what the rounding to T left over, rounded itself
__device__ __forceinline__ void store_rows(bf16_t* row, bf16_t* lo, const f32x16_t& v, float scale, int c0, int d, int lane, bool ok) {
#pragma unroll
  for (int pair = 0; pair < 2; ++pair) {
    uint32_t w[4], x[4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f0 = v[8 * pair + 4 * i + 2 * e] * scale, f1 = v[8 * pair + 4 * i + 2 * e + 1] * scale;
        w[2 * i + e] = f2bf_pk(f0, f1);
        x[2 * i + e] = lo != nullptr ? f2bf_pk(f0 - __uint_as_float(w[2 * i + e] << 16), f1 - __uint_as_float(w[2 * i + e] & 0xffff0000u)) : 0u;
      }
    swap_halves(w[0], w[2]);
    swap_halves(w[1], w[3]);
    const int c = c0 + 16 * pair + 8 * (lane >> 5);
    if (ok && c < d) *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
    if (lo != nullptr) {
      swap_halves(x[0], x[2]);
      swap_halves(x[1], x[3]);
      if (ok && c < d) *reinterpret_cast<uint4*>(lo + c) = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
}
__device__ __forceinline__ void store_rows(float* row, float*, const f32x16_t& v, float scale, int c0, int d, int lane, bool ok) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + 8 * i + 4 * (lane >> 5);
    if (ok && c < d) *reinterpret_cast<float4*>(row + c) = make_float4(v[4 * i] * scale, v[4 * i + 1] * scale, v[4 * i + 2] * scale, v[4 * i + 3] * scale);
  }
}

// One wave a SIMD has 256 ordinary and 256 accumulation registers.  The matrix instructions take their sums from either, but where values meet (the
// loop, the skipped tiles) the compiler wants ordinary ones: without this it moved 128 of them there and back in every tile.
template <bool ONE_WAVE, int N> __device__ __forceinline__ void accumulators(f32x16_t (&a)[N]) {
  if constexpr (ONE_WAVE) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+a"(a[i]));
  }
}

// Tiles of each kind in LDS.  A lone wave's LDS instructions run in order, so it overwrites a tile behind its own reads, and half the LDS lets more waves
// share a unit (captions of 5 .. 77 tokens, 21 k rows, forward: bf16 26.9 -> 24.3 us, float32 65.6 -> 50.8 us; training 107 -> 105, 248 -> 227 us).
constexpr int stages(int waves) { return waves == 1 ? 1 : 2; }

// The softmax statistics that the backward pass takes up: one number a query, its maximum + log2 of its sum; in float32 the two by themselves where the caller has
// room for them.  Their sum is rounded by 2^-24 of the maximum, which is an error of all probabilities of the query: with scores of 4096 dv was 4.7e-5 of its norm
// off, with the two numbers 4.4e-6 (32-bit elementary operations: 3.1e-6), for 0 .. 2 % of a training pass.  (To the 8 bits of a bf16 probability it is nothing.)
template <typename T> constexpr int statistics = sizeof(T) == 4 ? 3 : 2;  // of a query in the dk / dv kernel's LDS, with delta
template <typename T> __device__ __forceinline__ float* log_sums(const PA& p) { return sizeof(T) == 4 ? reinterpret_cast<float*>(p.out_lo) : nullptr; }

struct Item {
  int seq, block, head, start, len;
};
// work item of this workgroup.  Blocks are dealt out tile by tile with the heads fastest: when the head count is a multiple of the 8 XCDs (block
// b runs on XCD b % 8) neighbouring heads - the query heads of one key head - stay on one XCD and share its L2.
__device__ __forceinline__ Item work_item(const PA& p, int heads) {
  const int slot = blockIdx.x % heads, tile = blockIdx.x / heads;
  Item w;
  w.head = heads % 8 == 0 ? (slot & 7) * (heads >> 3) + (slot >> 3) : slot;
  const int* list = p.plan + ((p.seqs + 2) & ~1);
  w.seq = __builtin_amdgcn_readfirstlane(list[2 * tile]);
  w.block = __builtin_amdgcn_readfirstlane(list[2 * tile + 1]);
  w.start = __builtin_amdgcn_readfirstlane(w.seq >= 0 ? p.plan[w.seq] : p.plan[p.seqs]);
  w.len = __builtin_amdgcn_readfirstlane(w.seq >= 0 ? p.plan[w.seq + 1] : p.rows) - w.start;
  return w;
}
// rows behind the last sequence: zeros
template <typename T> __device__ __forceinline__ void zero_rows(T* base, long long row_stride, int r0, int n, int d, int tid, int nt) {
  constexpr int VN = Chunk<T>::N;
  const int ch = d / VN;
  for (int i = tid; i < n * ch; i += nt)
    *reinterpret_cast<uint4*>(base + (long long)(r0 + i / ch) * row_stride + (i % ch) * VN) = make_uint4(0, 0, 0, 0);
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// forward: workgroup = NW x 32 consecutive queries of one (sequence, query head)
// -----------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int CP, int NW, int KB, int OCC> __global__ __launch_bounds__(64 * NW, OCC) void packed_attn_fwd_kernel(PA p) {
  constexpr int PT = Tile<T, CP>::PT, NF = CP / 32, NK = CP / 16, NB = KB / 32, NT = 64 * NW, ST = stages(NW);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* const Kl = reinterpret_cast<T*>(smem);  // [ST][KB][PT]
  T* const Vl = Kl + ST * KB * PT;           // [ST][KB][PT]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item w = work_item(p, p.heads_q);
  if (w.seq < -1) return;
  T* const out = reinterpret_cast<T*>(p.out) + w.head * p.o_head;
  const int first = w.block * (32 * NW);
  if (w.seq < 0) {
    zero_rows(out + (long long)w.start * p.o_row, p.o_row, first, min(32 * NW, w.len - first), p.d, tid, NT);
    return;
  }
  const int q0 = first + wave * 32, my_q = q0 + (lane & 31);
  const bool q_ok = my_q < w.len;
  const int kv_head = w.head / (p.heads_q / p.heads_kv);
  const T* const qb = reinterpret_cast<const T*>(p.q) + (long long)w.start * p.q_row + w.head * p.q_head;
  const T* const kb = reinterpret_cast<const T*>(p.k) + (long long)w.start * p.k_row + kv_head * p.k_head;
  const T* const vb = reinterpret_cast<const T*>(p.v) + (long long)w.start * p.v_row + kv_head * p.v_head;
  const int keys = p.causal ? min(w.len, first + 32 * NW) : w.len;
  const int tiles = (keys + KB - 1) / KB;

  RowTile<T, CP, KB, NT> kt, vt;
  kt.place(p.k_row, p.d, tid);
  vt.place(p.v_row, p.d, tid);
  kt.start(kb, p.k_row, 0, w.len, p.d);
  vt.start(vb, p.v_row, 0, w.len, p.d);
  const Tile<T, CP> tile(lane);
  auto request = [&]() {
    kt.load();
    vt.load();
  };
  request();
  Frag<T> qf[NK];
  {
    const rsrc_t r = tile_rows(qb, p.q_row, q0, w.len, p.d);
    const int offset = (lane & 31) * (int)p.q_row * (int)sizeof(T);
#pragma unroll
    for (int k = 0; k < NK; ++k) qf[k] = gfrag(r, offset, 16 * k + 8 * (lane >> 5), p.d, qb);
  }
  kt.store(Kl, tid);
  vt.store(Vl, tid);
  request();

  const float c = p.scale * kL2E;  // scores in powers of two: exp(x) is one v_exp_f32
  float m = -INFINITY, l = 0.f;    // running maximum (of the unscaled scores) and sum
  f32x16_t o[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) o[f] = acc_zero();

  for (int t = 0; t < tiles; ++t) {
    const int k0 = t * KB;
    wg_barrier_lds();  // tile t is in LDS; everyone is done with tile t - 1, whose buffer tile t + 1 goes into
    const T* const Kt = Kl + t % ST * KB * PT;
    const T* const Vt = Vl + t % ST * KB * PT;
    auto advance = [&]() {
      kt.store(Kl + (t + 1) % ST * KB * PT, tid);
      vt.store(Vl + (t + 1) % ST * KB * PT, tid);
      request();
    };
    if (ST > 1) advance();
    if (NW > 1 && p.causal && k0 > q0 + 31) continue;  // in the future of all of this wave's queries
    f32x16_t s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = acc_zero();
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
      for (int b = 0; b < NB; ++b) mma32(s[b], tile.rows(Kt, 32 * b, 16 * k), qf[k]);
    if (k0 + KB > w.len || (p.causal && k0 + KB - 1 > q0)) {
      const int last = (p.causal ? min(my_q, w.len - 1) : w.len - 1) - k0 - 4 * (lane >> 5);  // the last key this lane's query sees, from its first row
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 32 * b + (r & 3) + 8 * (r >> 2) > last ? -INFINITY : s[b][r];
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
    // key 0 is visible to every query (and to the rows past the end, which count as zeros), so the maximum is finite from the first tile on
    // The reference point moves when a query's maximum is more than 2^8 past it: probabilities up to 2^8 instead of 1 have the same relative rounding, and
    // l and o stay far from float32's range; moved with every new maximum, half of the tiles scale o, 16 d / 32 multiplications (see above).
    // Per query, so that no result depends on the other queries of its wave.  (The negation: the first tile's -inf, and NaN, move.)
    const float m_new = fmaxf(m, both_halves_max(mx));
    const bool move = !((m_new - m) * c <= 8.f);
    if (__any(move)) {
      const float to = move ? m_new : m, alpha = pexp2((m - to) * c);
      l *= alpha;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[f][r] *= alpha;
      m = to;
    }
    const float mc = m * c;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = pexp2(fmaf(s[b][r], c, -mc));
        sum += s[b][r];
      }
    l += sum;  // this lane's half of the keys; the halves are joined once, at the end
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (b > 0 && p.causal && k0 + 32 * b > q0 + 31) continue;  // all zeros; and 0 times a NaN of the future would not be
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Frag<T> pf = acc_frag<T>(s[b], h);
#pragma unroll
        for (int f = 0; f < NF; ++f) mma32(o[f], tile.cols(Vt, 32 * b + 16 * h, 32 * f), pf);
      }
    }
    if (ST == 1) advance();
  }
  l = both_halves_sum(l);
  const float inv = 1.0f / l;
  const long long row = w.start + (q_ok ? my_q : 0);
  T* const lo = sizeof(T) == 2 && p.out_lo != nullptr ? reinterpret_cast<T*>(p.out_lo) + w.head * p.o_head + row * p.o_row : nullptr;
#pragma unroll
  for (int f = 0; f < NF; ++f) store_rows(out + row * p.o_row, lo, o[f], inv, 32 * f, p.d, lane, q_ok);
  if (lane < 32 && q_ok && p.lse != nullptr) {
    const long long at = (long long)w.head * p.rows + row;
    float* const sums = log_sums<T>(p);
    p.lse[at] = sums != nullptr ? m * c : fmaf(m, c, __log2f(l));
    if (sums != nullptr) sums[at] = __log2f(l);
  }
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// backward, dq (and delta): workgroup = NW x 32 consecutive queries of one (sequence, query head)
// -----------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int CP, int NW, int KB, int OCC> __global__ __launch_bounds__(64 * NW, OCC) void packed_attn_dq_kernel(PA p) {
  constexpr int PT = Tile<T, CP>::PT, NF = CP / 32, NK = CP / 16, NB = KB / 32, NT = 64 * NW, ST = stages(NW);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* const Kl = reinterpret_cast<T*>(smem);
  T* const Vl = Kl + ST * KB * PT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item w = work_item(p, p.heads_q);
  if (w.seq < -1) return;
  T* const dq = reinterpret_cast<T*>(p.dq) + w.head * p.dq_head;
  const int first = w.block * (32 * NW);
  if (w.seq < 0) {
    zero_rows(dq + (long long)w.start * p.dq_row, p.dq_row, first, min(32 * NW, w.len - first), p.d, tid, NT);
    return;
  }
  const int q0 = first + wave * 32, my_q = q0 + (lane & 31);
  const bool q_ok = my_q < w.len;
  const int kv_head = w.head / (p.heads_q / p.heads_kv);
  const T* const qb = reinterpret_cast<const T*>(p.q) + (long long)w.start * p.q_row + w.head * p.q_head;
  const T* const db = reinterpret_cast<const T*>(p.dout) + (long long)w.start * p.do_row + w.head * p.do_head;
  const T* const ob = reinterpret_cast<const T*>(p.out) + (long long)w.start * p.o_row + w.head * p.o_head;
  const bool two = sizeof(T) == 2 && p.out_lo != nullptr;
  const T* const lb = reinterpret_cast<const T*>(two ? p.out_lo : p.out) + (long long)w.start * p.o_row + w.head * p.o_head;
  const T* const kb = reinterpret_cast<const T*>(p.k) + (long long)w.start * p.k_row + kv_head * p.k_head;
  const T* const vb = reinterpret_cast<const T*>(p.v) + (long long)w.start * p.v_row + kv_head * p.v_head;
  const int keys = p.causal ? min(w.len, first + 32 * NW) : w.len;
  const int tiles = (keys + KB - 1) / KB;

  RowTile<T, CP, KB, NT> kt, vt;
  kt.place(p.k_row, p.d, tid);
  vt.place(p.v_row, p.d, tid);
  kt.start(kb, p.k_row, 0, w.len, p.d);
  vt.start(vb, p.v_row, 0, w.len, p.d);
  const Tile<T, CP> tile(lane);
  auto request = [&]() {
    kt.load();
    vt.load();
  };
  request();
  Frag<T> qf[NK], df[NK];
  float delta = 0.f;
  {
    const rsrc_t rq = tile_rows(qb, p.q_row, q0, w.len, p.d), rd = tile_rows(db, p.do_row, q0, w.len, p.d), ro = tile_rows(ob, p.o_row, q0, w.len, p.d);
    const rsrc_t rl = two ? tile_rows(lb, p.o_row, q0, w.len, p.d) : rows_of(lb, 0);
    const int r = (lane & 31) * (int)sizeof(T), oq = r * (int)p.q_row, od = r * (int)p.do_row, oo = r * (int)p.o_row;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int c0 = 16 * k + 8 * (lane >> 5);
      qf[k] = gfrag(rq, oq, c0, p.d, qb);
      df[k] = gfrag(rd, od, c0, p.d, qb);
      delta += frag_dot(df[k], gfrag(ro, oo, c0, p.d, qb)) + frag_dot(df[k], gfrag(rl, oo, c0, p.d, qb));
    }
  }
  delta = both_halves_sum(delta);
  const long long row = w.start + (q_ok ? my_q : 0), at = (long long)w.head * p.rows + row;
  const float* const sums = log_sums<T>(p);
  const float lse = p.lse[at], log_sum = sums != nullptr ? sums[at] : 0.f;
  if (lane < 32 && q_ok) p.delta[at] = delta;  // read by the dk / dv kernel behind this one
  kt.store(Kl, tid);
  vt.store(Vl, tid);
  request();
  const float c = p.scale * kL2E;
  f32x16_t acc[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) acc[f] = acc_zero();

  f32x16_t minus_delta;  // the products with V start from it
#pragma unroll
  for (int r = 0; r < 16; ++r) minus_delta[r] = -delta;
  for (int t = 0; t < tiles; ++t) {
    const int k0 = t * KB;
    accumulators<OCC == 1>(acc);
    wg_barrier_lds();
    const T* const Kt = Kl + t % ST * KB * PT;
    const T* const Vt = Vl + t % ST * KB * PT;
    auto advance = [&]() {
      kt.store(Kl + (t + 1) % ST * KB * PT, tid);
      vt.store(Vl + (t + 1) % ST * KB * PT, tid);
      request();
    };
    if (ST > 1) advance();
    if (NW > 1 && p.causal && k0 > q0 + 31) continue;
    const bool masked = k0 + KB > w.len || (p.causal && k0 + KB - 1 > q0);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (b > 0 && p.causal && k0 + 32 * b > q0 + 31) continue;  // (as in the forward)
      f32x16_t s = acc_zero(), dp = minus_delta;
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        mma32(s, tile.rows(Kt, 32 * b, 16 * k), qf[k]);
        mma32(dp, tile.rows(Vt, 32 * b, 16 * k), df[k]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = pexp2(sizeof(T) == 4 ? fmaf(s[r], c, -lse) - log_sum : fmaf(s[r], c, -lse)) * dp[r];
      if (masked) {
        const int last = (p.causal ? min(my_q, w.len - 1) : w.len - 1) - k0 - 32 * b - 4 * (lane >> 5);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (r & 3) + 8 * (r >> 2) > last ? 0.f : s[r];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Frag<T> sf = acc_frag<T>(s, h);
#pragma unroll
        for (int f = 0; f < NF; ++f) mma32(acc[f], tile.cols(Kt, 32 * b + 16 * h, 32 * f), sf);
      }
    }
    if (ST == 1) advance();
  }
  accumulators<OCC == 1>(acc);
#pragma unroll
  for (int f = 0; f < NF; ++f) store_rows(dq + row * p.dq_row, (T*)nullptr, acc[f], p.scale, 32 * f, p.d, lane, q_ok);
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// backward, dk and dv: workgroup = NW x 32 consecutive keys of one (sequence, key head); loops over the group's query heads and the queries
// -----------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int CP, int NW, int QB, int OCC> __global__ __launch_bounds__(64 * NW, OCC) void packed_attn_dkv_kernel(PA p) {
  constexpr int PT = Tile<T, CP>::PT, NF = CP / 32, NK = CP / 16, NB = QB / 32, NT = 64 * NW, ST = stages(NW);
  // 32-query blocks whose scores are held at once: a lone wave has nothing else to put under their MFMAs (96 and 128 columns: 2 % off the pass)
  constexpr int SB = OCC == 1 ? NB : 1;
  static_assert(NT >= QB, "one thread a query's statistics");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* const Ql = reinterpret_cast<T*>(smem);
  T* const Dl = Ql + ST * QB * PT;
  constexpr int NL = statistics<T>;
  float* const Ll = reinterpret_cast<float*>(Dl + ST * QB * PT);  // [ST][NL][NT]: log-sums (maxima), -deltas, (log-sums) of a tile's queries
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item w = work_item(p, p.heads_kv);
  if (w.seq < -1) return;
  T* const dk = reinterpret_cast<T*>(p.dk) + w.head * p.dk_head;
  T* const dv = reinterpret_cast<T*>(p.dv) + w.head * p.dv_head;
  // the list has the blocks with the most keys in front of them first; a key block's cost is the queries BEHIND it: read the list mirrored
  const int first = w.seq < 0 ? w.block * (32 * NW) : ((w.len + 32 * NW - 1) / (32 * NW) - 1 - w.block) * (32 * NW);
  if (w.seq < 0) {
    zero_rows(dk + (long long)w.start * p.dk_row, p.dk_row, first, min(32 * NW, w.len - first), p.d, tid, NT);
    zero_rows(dv + (long long)w.start * p.dv_row, p.dv_row, first, min(32 * NW, w.len - first), p.d, tid, NT);
    return;
  }
  const int k0 = first + wave * 32, my_k = k0 + (lane & 31);
  const bool k_ok = my_k < w.len;
  const int group = p.heads_q / p.heads_kv;
  const T* const kb = reinterpret_cast<const T*>(p.k) + (long long)w.start * p.k_row + w.head * p.k_head;
  const T* const vb = reinterpret_cast<const T*>(p.v) + (long long)w.start * p.v_row + w.head * p.v_head;
  const int qfirst = p.causal ? first : 0;
  const int per_head = (w.len - qfirst + QB - 1) / QB, tiles = group * per_head;

  RowTile<T, CP, QB, NT> qt, dt;
  qt.place(p.q_row, p.d, tid);
  dt.place(p.do_row, p.d, tid);
  const Tile<T, CP> tile(lane);
  float lse, delta, log_sum = 0.f;
  const float* const sums = log_sums<T>(p);
  int next_head = w.head * group, next_q = w.len;  // of the tile that is requested next; behind a head's last one: start the next head
  const int end_head = next_head + group, offset = tid < QB ? tid * 4 : kBeyond;
  auto request = [&]() {
    if (next_q >= w.len) {
      const int head = min(next_head, end_head - 1), len = next_head < end_head ? w.len : qfirst;  // (behind the last head: nothing)
      qt.start(reinterpret_cast<const T*>(p.q) + (long long)w.start * p.q_row + head * p.q_head, p.q_row, qfirst, len, p.d);
      dt.start(reinterpret_cast<const T*>(p.dout) + (long long)w.start * p.do_row + head * p.do_head, p.do_row, qfirst, len, p.d);
      if (next_head < end_head) next_q = qfirst;
      ++next_head;
    }
    qt.load();
    dt.load();
    const long long at = (long long)min(next_head - 1, end_head - 1) * p.rows + w.start + next_q;
    const long long bytes = next_head <= end_head ? (long long)(w.len - next_q) * 4 : 0;
    lse = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows_of(p.lse + at, bytes), offset, 0, 0));
    delta = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows_of(p.delta + at, bytes), offset, 0, 0));
    if (sizeof(T) == 4) log_sum = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows_of(sums + (sums != nullptr ? at : 0), sums != nullptr ? bytes : 0), offset, 0, 0));
    next_q += QB;
  };
  auto store = [&](int t) {
    qt.store(Ql + t % ST * QB * PT, tid);
    dt.store(Dl + t % ST * QB * PT, tid);
    Ll[t % ST * NL * NT + tid] = lse;
    Ll[t % ST * NL * NT + NT + tid] = -delta;
    if (NL == 3) Ll[t % ST * NL * NT + 2 * NT + tid] = log_sum;
  };
  request();
  Frag<T> kf[NK], vf[NK];
  {
    const rsrc_t rk = tile_rows(kb, p.k_row, k0, w.len, p.d), rv = tile_rows(vb, p.v_row, k0, w.len, p.d);
    const int r = (lane & 31) * (int)sizeof(T);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      kf[k] = gfrag(rk, r * (int)p.k_row, 16 * k + 8 * (lane >> 5), p.d, kb);
      vf[k] = gfrag(rv, r * (int)p.v_row, 16 * k + 8 * (lane >> 5), p.d, kb);
    }
  }
  store(0);
  request();

  const float c = p.scale * kL2E;
  f32x16_t ak[NF], av[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) { ak[f] = acc_zero(); av[f] = acc_zero(); }

  for (int t = 0, q0 = qfirst; t < tiles; ++t, q0 = q0 + QB < w.len ? q0 + QB : qfirst) {
    accumulators<OCC == 1>(ak);
    accumulators<OCC == 1>(av);
    wg_barrier_lds();
    auto advance = [&]() {
      store(t + 1);
      request();
    };
    if (ST > 1) advance();
    const T* const Qt = Ql + t % ST * QB * PT;
    const T* const Dt = Dl + t % ST * QB * PT;
    const float* const Lt = Ll + t % ST * NL * NT;
    if (NW > 1 && (k0 >= w.len || (p.causal && q0 + QB - 1 < k0))) continue;  // no key of this wave, or none of the tile's queries sees one
    const bool masked = q0 + QB > w.len || (p.causal && q0 < k0 + 31);
#pragma unroll
    for (int b0 = 0; b0 < NB; b0 += SB) {
      if (SB == 1 && b0 + 1 < NB && p.causal && q0 + 32 * b0 + 31 < k0) continue;  // none of these queries sees a key of this wave
      f32x16_t s[SB], dp[SB];  // dp starts from -delta
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        s[b] = acc_zero();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 de = *reinterpret_cast<const float4*>(Lt + NT + 32 * (b0 + b) + 8 * i + 4 * (lane >> 5));
          dp[b][4 * i] = de.x; dp[b][4 * i + 1] = de.y; dp[b][4 * i + 2] = de.z; dp[b][4 * i + 3] = de.w;
        }
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          mma32(s[b], tile.rows(Qt, 32 * (b0 + b), 16 * k), kf[k]);
          mma32(dp[b], tile.rows(Dt, 32 * (b0 + b), 16 * k), vf[k]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 ls = *reinterpret_cast<const float4*>(Lt + 32 * (b0 + b) + 8 * i + 4 * (lane >> 5));
          const float lv[4] = {ls.x, ls.y, ls.z, ls.w};
          float4 lg = make_float4(0.f, 0.f, 0.f, 0.f);
          if (NL == 3) lg = *reinterpret_cast<const float4*>(Lt + 2 * NT + 32 * (b0 + b) + 8 * i + 4 * (lane >> 5));
          const float gv[4] = {lg.x, lg.y, lg.z, lg.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = fmaf(s[b][4 * i + e], c, -lv[e]);
            s[b][4 * i + e] = pexp2(NL == 3 ? x - gv[e] : x);
            dp[b][4 * i + e] *= s[b][4 * i + e];
          }
        }
      }
      if (masked) {
#pragma unroll
        for (int b = 0; b < SB; ++b) {
          // queries from `lo` on (from this lane's first row) see this lane's key, those from `hi` on lie behind the sequence
          const int base = q0 + 32 * (b0 + b) + 4 * (lane >> 5), lo = p.causal ? my_k - base : -64, hi = w.len - base;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int q = (r & 3) + 8 * (r >> 2);
            const bool hide = q < lo || q >= hi;
            s[b][r] = hide ? 0.f : s[b][r];
            dp[b][r] = hide ? 0.f : dp[b][r];
          }
        }
      }
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        if (b + 1 < SB && p.causal && q0 + 32 * b + 31 < k0) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Frag<T> pf = acc_frag<T>(s[b], h), sf = acc_frag<T>(dp[b], h);
#pragma unroll
          for (int f = 0; f < NF; ++f) {
            mma32(av[f], tile.cols(Dt, 32 * (b0 + b) + 16 * h, 32 * f), pf);
            mma32(ak[f], tile.cols(Qt, 32 * (b0 + b) + 16 * h, 32 * f), sf);
          }
        }
      }
    }
    if (ST == 1) advance();
  }
  accumulators<OCC == 1>(ak);
  accumulators<OCC == 1>(av);
  const long long row = w.start + (k_ok ? my_k : 0);
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    store_rows(dk + row * p.dk_row, (T*)nullptr, ak[f], p.scale, 32 * f, p.d, lane, k_ok);
    store_rows(dv + row * p.dv_row, (T*)nullptr, av[f], 1.f, 32 * f, p.d, lane, k_ok);
  }
}

// -----------------------------------------------------------------------------------------------------------------------------------------
// plan: starts[0 .. seqs] (from 0, clamped into 0 .. rows and made monotone, so that no kernel can be led out of its buffers), then the list of
// (sequence, block) pairs by falling block index, the filling blocks behind the last sequence as (-1, block), and (-2, 0) for unused places.
// One workgroup; LDS counters give the places, whose order among equals does not matter (every item's results are its own).
// -----------------------------------------------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024, kClasses = 512;
__global__ __launch_bounds__(kPlanThreads) void packed_plan_kernel(const int* __restrict__ cu, int seqs, int rows, int block, int* __restrict__ plan, int places) {
  __shared__ int part[kPlanThreads];
  __shared__ int count[kClasses], place[kClasses];
  const int tid = threadIdx.x;
  // starts: running maximum over chunks of consecutive entries
  const int n = seqs + 1, per = (n + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * per, n), i1 = min(i0 + per, n);
  auto boundary = [&](int i) { return i ? min(max(cu[i], 0), rows) : 0; };  // (the first one counts as 0: no row is without an owner)
  int top = 0;
  for (int i = i0; i < i1; ++i) top = max(top, boundary(i));
  part[tid] = top;
  for (int c = tid; c < kClasses; c += kPlanThreads) count[c] = 0;
  __syncthreads();
  for (int o = 1; o < kPlanThreads; o <<= 1) {
    const int v = tid >= o ? part[tid - o] : 0;
    __syncthreads();
    part[tid] = max(part[tid], v);
    __syncthreads();
  }
  int run = tid ? part[tid - 1] : 0;
  for (int i = i0; i < i1; ++i) {
    run = max(run, boundary(i));
    plan[i] = run;
  }
  __threadfence_block();
  __syncthreads();
  const int lane = tid & 63, wave = tid >> 6;
  for (int s = wave; s < seqs; s += kPlanThreads / 64) {
    const int nb = (plan[s + 1] - plan[s] + block - 1) / block;
    for (int b = lane; b < nb; b += 64) atomicAdd(&count[min(b, kClasses - 1)], 1);
  }
  __syncthreads();
  part[tid] = tid < kClasses ? count[kClasses - 1 - tid] : 0;
  __syncthreads();
  for (int o = 1; o < kClasses; o <<= 1) {
    const int v = tid >= o ? part[tid - o] : 0;
    __syncthreads();
    part[tid] += v;
    __syncthreads();
  }
  if (tid < kClasses) place[kClasses - 1 - tid] = tid ? part[tid - 1] : 0;
  __syncthreads();
  const int used = part[kClasses - 1];
  int* const list = plan + ((seqs + 2) & ~1);
  for (int s = wave; s < seqs; s += kPlanThreads / 64) {
    const int nb = (plan[s + 1] - plan[s] + block - 1) / block;
    for (int b = lane; b < nb; b += 64) {
      const int at = atomicAdd(&place[min(b, kClasses - 1)], 1);
      list[2 * at] = s;
      list[2 * at + 1] = b;
    }
  }
  const int tail = (rows - plan[seqs] + block - 1) / block;
  for (int i = used + tid; i < places; i += kPlanThreads) {
    list[2 * i] = i < used + tail ? -1 : -2;
    list[2 * i + 1] = i < used + tail ? i - used : 0;
  }
}

// waves per SIMD that the register budget is set for: 2, and 1 where a lone wave stages wide tiles by itself or the accumulators are many
template <typename T, int CP, int NW> constexpr int occ(bool two_accumulators) {
  return NW == 1 ? (CP > 64 || (sizeof(T) == 4 && CP > 32) ? 1 : 2) : two_accumulators && (CP > 64 || (sizeof(T) == 4 && CP > 32)) ? 1 : sizeof(T) == 4 && CP > 64 ? 1 : 2;
}
template <typename T, int CP, int NW, int KB> int launch_fwd(const PA& p, hipStream_t st) {
  constexpr auto kernel = packed_attn_fwd_kernel<T, CP, NW, KB, occ<T, CP, NW>(false)>;
  static DynSmemAttr attr;
  const size_t smem = (size_t)2 * stages(NW) * KB * Tile<T, CP>::PT * sizeof(T);
  if (hipError_t e = attr.ensure((const void*)kernel, smem)) return (int)e;
  kernel<<<dim3((unsigned)(p.places * p.heads_q)), dim3(64 * NW), smem, st>>>(p);
  CVH_CHECK_LAUNCH();
  return 0;
}
template <typename T, int CP, int NW, int KB> int launch_bwd(const PA& p, hipStream_t st) {
  constexpr int QB = sizeof(T) == 2 && NW == 4 ? 64 : KB;
  constexpr auto dq = packed_attn_dq_kernel<T, CP, NW, KB, occ<T, CP, NW>(false)>;
  constexpr auto dkv = packed_attn_dkv_kernel<T, CP, NW, QB, occ<T, CP, NW>(true)>;
  static DynSmemAttr aq, ak;
  constexpr int tiles = 2 * stages(NW);
  const size_t sq = (size_t)tiles * KB * Tile<T, CP>::PT * sizeof(T), sk = (size_t)tiles * QB * Tile<T, CP>::PT * sizeof(T) + stages(NW) * statistics<T> * 64 * NW * sizeof(float);
  if (hipError_t e = aq.ensure((const void*)dq, sq)) return (int)e;
  if (hipError_t e = ak.ensure((const void*)dkv, sk)) return (int)e;
  dq<<<dim3((unsigned)(p.places * p.heads_q)), dim3(64 * NW), sq, st>>>(p);
  dkv<<<dim3((unsigned)(p.places * p.heads_kv)), dim3(64 * NW), sk, st>>>(p);
  CVH_CHECK_LAUNCH();
  return 0;
}
template <typename T, int CP> int run_width(const PA& p, int backward, hipStream_t st) {
  constexpr int KB4 = sizeof(T) == 2 && CP <= 64 ? 64 : 32;
  if (p.block == 32) return backward ? launch_bwd<T, CP, 1, 32>(p, st) : launch_fwd<T, CP, 1, 32>(p, st);
  return backward ? launch_bwd<T, CP, 4, KB4>(p, st) : launch_fwd<T, CP, 4, sizeof(T) == 2 ? 64 : 32>(p, st);
}
template <typename T> int run_type(const PA& p, int backward, hipStream_t st) {
  switch ((p.d + 31) / 32) {
    case 1: return run_width<T, 32>(p, backward, st);
    case 2: return run_width<T, 64>(p, backward, st);
    case 3: return run_width<T, 96>(p, backward, st);
    default: return run_width<T, 128>(p, backward, st);
  }
}

constexpr int kMostRows = 0x7fffffff - 4096;  // and sequences: blocks are counted in 32 bits
bool strides_ok(int dtype, const void* base, long long row, long long head) {
  const long long n = dtype == CVH_DT_BF16 ? 8 : 4;  // 16-byte accesses
  return base != nullptr && (reinterpret_cast<uintptr_t>(base) & 15) == 0 && row % n == 0 && head % n == 0 && row >= 0 && head >= 0 && row <= (1 << 21);  // (128 rows in 31 bits of bytes)
}
int check(int dtype, const PA* p, int backward) {
  if (dtype != CVH_DT_F32 && dtype != CVH_DT_BF16) return -1;
  if (p == nullptr || p->plan == nullptr) return -2;
  if (p->rows <= 0 || p->rows > kMostRows || p->seqs <= 0 || p->seqs > kMostRows || p->heads_q <= 0 || p->heads_kv <= 0 || p->heads_q % p->heads_kv || p->d <= 0 || p->d > 128 || p->d % 8) return -2;
  if (!(p->scale > 0.f) || (p->block != 32 && p->block != 128)) return -2;
  if (p->places != (long long)p->rows / p->block + p->seqs + 1 || (long long)p->places * p->heads_q >= (1 << 24)) return -2;  // (a grid has fewer than 2^32 threads)
  if (!strides_ok(dtype, p->q, p->q_row, p->q_head) || !strides_ok(dtype, p->k, p->k_row, p->k_head) || !strides_ok(dtype, p->v, p->v_row, p->v_head) ||
      !strides_ok(dtype, p->out, p->o_row, p->o_head))
    return -2;
  if (p->out_lo != nullptr && (reinterpret_cast<uintptr_t>(p->out_lo) & 15)) return -2;
  if (backward && (p->lse == nullptr || p->delta == nullptr || !strides_ok(dtype, p->dout, p->do_row, p->do_head) || !strides_ok(dtype, p->dq, p->dq_row, p->dq_head) ||
                   !strides_ok(dtype, p->dk, p->dk_row, p->dk_head) || !strides_ok(dtype, p->dv, p->dv_row, p->dv_head)))
    return -2;
  return 0;
}

}  // namespace

extern "C" long long cvh_packed_plan_elems(int seqs, int rows, int block) {
  if (seqs <= 0 || seqs > kMostRows || rows <= 0 || rows > kMostRows || (block != 32 && block != 128)) return -2;
  return ((long long)(seqs + 2) & ~1ll) + 2 * ((long long)rows / block + seqs + 1);
}
extern "C" int cvh_packed_plan(const int* cu, int seqs, int rows, int block, int* plan, void* stream) {
  if (cu == nullptr || plan == nullptr || seqs <= 0 || seqs > kMostRows || rows <= 0 || rows > kMostRows || (block != 32 && block != 128)) return -2;
  if ((long long)rows / block + seqs + 1 >= 1 << 24) return -2;  // more than any launch over the list takes
  hipLaunchKernelGGL(packed_plan_kernel, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, cu, seqs, rows, block, plan, rows / block + seqs + 1);
  CVH_CHECK_LAUNCH();
  return 0;
}
extern "C" int cvh_packed_attn_fwd(int dtype, const cvh_packed_attn* p, void* stream) {
  if (int rc = check(dtype, p, 0)) return rc;
  return dtype == CVH_DT_BF16 ? run_type<bf16_t>(*p, 0, (hipStream_t)stream) : run_type<float>(*p, 0, (hipStream_t)stream);
}
extern "C" int cvh_packed_attn_bwd(int dtype, const cvh_packed_attn* p, void* stream) {
  if (int rc = check(dtype, p, 1)) return rc;
  return dtype == CVH_DT_BF16 ? run_type<bf16_t>(*p, 1, (hipStream_t)stream) : run_type<float>(*p, 1, (hipStream_t)stream);
}
