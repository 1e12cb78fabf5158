// Token embedding on packed rows and its gradient by sorted tokens.
//
//   y_r = scale * table[id_r] + pos[r - cu[seq(r)]]
//   dtable[v] = scale * sum over { r : id_r = v } of dy_r, in the order of r;     dpos[t] = sum over the sequences b longer than t of dy[cu_b + t]
//
// The gradient of the table is dense float32.  Scattering with float atomics makes its sums depend on the order in which they retire and needs
// the table zeroed first; here the rows are sorted by token (stable radix sort, 8 bits a pass), every row of the table is then written exactly
// once, as the sum of its run in a fixed order: bit-reproducible.  What bounds it: the write of the whole table (49408 x 512: 101 MB) next to
// one read of dy.  A frequent token (the start mark of every caption) would leave its whole run to one wave: runs longer than kChunk are summed
// in pieces of kChunk rows first, by as many waves, and joined in order.
#include "common.hpp"
#include "cvnets_hip.h"

namespace {

constexpr int kItems = 2048;   // rows a sort workgroup takes: 4 waves x 8 rounds x 64 lanes
constexpr int kChunk = 64;     // rows of a piece
constexpr int kTableRows = 32;  // rows of the table a workgroup writes

// sort key of row r: its token, or `vocab` (sorted behind everything) where the row adds nothing: behind the last sequence, the padding token,
// a token outside the table
__device__ __forceinline__ unsigned token_key(const long long* ids, int r, const int* cu, int seqs, long long padding, int vocab) {
  const long long t = ids[r];
  const bool used = (cu == nullptr || r < cu[seqs]) && t >= 0 && t < vocab && t != padding;
  return used ? (unsigned)t : (unsigned)vocab;
}

struct SortIn {
  const long long* ids;  // first pass: tokens
  const int* starts;     // boundaries (plan of the layout) or null
  const unsigned* keys;  // later passes: the previous pass's keys and rows
  const int* rows;
  long long padding;
  int n, seqs, vocab, shift;
};
__device__ __forceinline__ unsigned sort_key(const SortIn& s, int i) {
  return s.keys != nullptr ? s.keys[i] : token_key(s.ids, i, s.starts, s.seqs, s.padding, s.vocab);
}

// digits of one workgroup's rows, counted: count[block][256]
__global__ __launch_bounds__(256) void sort_count_kernel(SortIn s, int* __restrict__ count) {
  __shared__ int c[256];
  c[threadIdx.x] = 0;
  __syncthreads();
  const int base = blockIdx.x * kItems;
  for (int i = threadIdx.x; i < kItems && base + i < s.n; i += 256) atomicAdd(&c[(sort_key(s, base + i) >> s.shift) & 255], 1);
  __syncthreads();
  count[blockIdx.x * 256 + threadIdx.x] = c[threadIdx.x];
}

// stable scatter of one pass.  A wave's rows are consecutive; a lane's place = rows of smaller digits + of this digit in earlier workgroups, waves
// and rounds + in lower lanes of its round (8 ballots find the lanes with the same digit).
__global__ __launch_bounds__(256) void sort_scatter_kernel(SortIn s, const int* __restrict__ count, unsigned* __restrict__ keys_out, int* __restrict__ rows_out) {
  __shared__ int at[4][256];  // counts, then next place, of each wave and digit
  __shared__ int scan[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int w = 0; w < 4; ++w) at[w][tid] = 0;
  __syncthreads();
  const int base = blockIdx.x * kItems + wave * (kItems / 4);
  unsigned key[kItems / 256];
#pragma unroll
  for (int j = 0; j < kItems / 256; ++j) {
    const int i = base + j * 64 + lane;
    key[j] = i < s.n ? sort_key(s, i) : 0u;
    if (i < s.n) atomicAdd(&at[wave][(key[j] >> s.shift) & 255], 1);
  }
  __syncthreads();
  int before = 0, total = 0;  // digit `tid`: rows in earlier workgroups, rows in all
  if (gridDim.x == 1) {
    total = at[0][tid] + at[1][tid] + at[2][tid] + at[3][tid];
  } else {
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int v = count[b * 256 + tid];
      before += b < (int)blockIdx.x ? v : 0;
      total += v;
    }
  }
  scan[tid] = total;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const int v = tid >= o ? scan[tid - o] : 0;
    __syncthreads();
    scan[tid] += v;
    __syncthreads();
  }
  int p = scan[tid] - total + before;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int v = at[w][tid];
    at[w][tid] = p;
    p += v;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems / 256; ++j) {
    const int i = base + j * 64 + lane;
    const bool in = i < s.n;
    const unsigned d = (key[j] >> s.shift) & 255;
    unsigned long long same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const unsigned long long one = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? one : ~one;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    int to = 0;
    if (in) to = at[wave][d] + rank;
    wave_lds_sync();
    if (in && rank == 0) at[wave][d] += __popcll(same);
    wave_lds_sync();
    if (in) {
      keys_out[to] = key[j];
      rows_out[to] = s.keys != nullptr ? s.rows[i] : i;
    }
  }
}

// first position in keys[lo .. hi) that holds a key >= v, by one wave: 64 probes a step
__device__ __forceinline__ int lower_bound_wave(const unsigned* keys, int lo, int hi, unsigned v, int lane) {
  while (hi - lo > 64) {
    const int step = (hi - lo + 64) / 65;
    const int at = lo + (lane + 1) * step - 1;  // probes; the answer lies behind the last one that is smaller
    const int below = __popcll(__ballot(at < hi && keys[min(at, hi - 1)] < v));
    const int nlo = lo + below * step;
    hi = below < 64 ? min(hi, nlo + step) : hi;
    lo = min(nlo, hi);
  }
  const int at = lo + lane;
  return lo + __popcll(__ballot(at < hi && keys[min(at, hi > lo ? hi - 1 : lo)] < v));
}
__device__ __forceinline__ int lower_bound_lane(const unsigned* keys, int lo, int hi, unsigned v) {
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// acc[0 .. 8) += columns c .. c + 7 of dy rows order[a .. b), in order; four rows in flight
template <typename T> __device__ __forceinline__ void add_rows(const T* __restrict__ dy, const int* __restrict__ order, int a, int b, int e, int c, float* acc) {
  int i = a;
  for (; i + 4 <= b; i += 4) {
    V8<T> v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = v8_load<T>(dy + (size_t)order[i + j] * e + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[8];
      v8_unpack(v[j], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += f[k];
    }
  }
  for (; i < b; ++i) {
    float f[8];
    v8_unpack(v8_load<T>(dy + (size_t)order[i] * e + c), f);
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] += f[k];
  }
}

// pieces of the long runs (more than kChunk rows): chunk c of the sorted rows has part[c][0] for the run its first row belongs to and part[c][1]
// for the run its last row belongs to, where that is another one.  One wave a chunk.
template <typename T>
__global__ __launch_bounds__(256) void embed_pieces_kernel(const T* __restrict__ dy, const unsigned* __restrict__ keys, const int* __restrict__ order, int n,
                                                           int vocab, int e, float* __restrict__ part) {
  const int lane = threadIdx.x & 63, chunk = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int a = chunk * kChunk, b = min(a + kChunk, n);
  if (a >= n) return;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const unsigned v = keys[side ? b - 1 : a];
    if (v >= (unsigned)vocab || (side && v == keys[a])) continue;
    // long: the run reaches at least kChunk + 1 rows; inside this chunk it is [lo, hi)
    const int from = max(0, a - kChunk), to = min(n, b + kChunk);
    const int lo = lower_bound_wave(keys, from, to, v, lane), hi = lower_bound_wave(keys, from, to, v + 1, lane);
    const bool is_long = hi - lo > kChunk || (lo == from && from > 0) || (hi == to && to < n);
    if (!is_long) continue;
    // (a run that only touches the window's end may still be short: the rows kernel decides by the run itself and then does not read this piece)
    for (int c = lane * 8; c < e; c += 512) {
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      add_rows<T>(dy, order, max(lo, a), min(hi, b), e, c, acc);
      float* p = part + ((size_t)chunk * 2 + side) * e + c;
      *reinterpret_cast<float4*>(p) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
  }
}

// rows v0 .. v0 + kTableRows - 1 of the gradient, each written once: zeros, the sum of a short run, or of a long run's pieces (by all four waves)
template <typename T>
__global__ __launch_bounds__(256) void embed_rows_kernel(const T* __restrict__ dy, const unsigned* __restrict__ keys, const int* __restrict__ order, int n,
                                                         int vocab, int e, float scale, const float* __restrict__ part, float* __restrict__ dtable, int group) {
  __shared__ int bound[kTableRows + 1];
  __shared__ int range[2];
  __shared__ __attribute__((aligned(16))) float joined[4][512];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int v0 = blockIdx.x * kTableRows, rows = min(kTableRows, vocab - v0);
  if (wave < 2) {
    const int at = lower_bound_wave(keys, 0, n, (unsigned)(wave ? v0 + rows : v0), lane);
    if (lane == 0) range[wave] = at;
  }
  __syncthreads();
  if (tid <= rows) bound[tid] = lower_bound_lane(keys, range[0], range[1], (unsigned)(v0 + tid));
  __syncthreads();
  const int per = 256 / group, sub = tid / group, sl = tid % group;  // `group` lanes a row
  for (int r = sub; r < rows; r += per) {
    const int a = bound[r], b = bound[r + 1];
    if (b - a > kChunk) continue;
    for (int c = sl * 8; c < e; c += group * 8) {
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      add_rows<T>(dy, order, a, b, e, c, acc);
      float* p = dtable + (size_t)(v0 + r) * e + c;
      *reinterpret_cast<float4*>(p) = make_float4(acc[0] * scale, acc[1] * scale, acc[2] * scale, acc[3] * scale);
      *reinterpret_cast<float4*>(p + 4) = make_float4(acc[4] * scale, acc[5] * scale, acc[6] * scale, acc[7] * scale);
    }
  }
  for (int r = 0; r < rows; ++r) {
    const int a = bound[r], b = bound[r + 1];
    if (b - a <= kChunk) continue;  // the same for the whole workgroup
    const int c0 = a / kChunk, c1 = (b - 1) / kChunk, first = a % kChunk ? 1 : 0;
    for (int base = 0; base < e; base += 512) {
      const int c = base + lane * 8;
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (c < e) {
#pragma unroll 4
        for (int k = c0 + wave; k <= c1; k += 4) {
          // (of the run's first chunk the piece is the one of its last row, unless the run begins with the chunk)
          const float* p = part + ((size_t)k * 2 + (k == c0 ? first : 0)) * e + c;
          const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
          acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
          acc[4] += y.x; acc[5] += y.y; acc[6] += y.z; acc[7] += y.w;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) joined[wave][lane * 8 + k] = acc[k];
      __syncthreads();
      for (int k = tid; k < 512 && base + k < e; k += 256)
        dtable[(size_t)(v0 + r) * e + base + k] = ((joined[0][k] + joined[1][k]) + (joined[2][k] + joined[3][k])) * scale;
      __syncthreads();
    }
  }
}

// one workgroup a position: the rows at that place of all sequences, 16 waves over the sequences, joined in order
template <typename T>
__global__ __launch_bounds__(1024) void embed_pos_kernel(const T* __restrict__ dy, const int* __restrict__ starts, int seqs, int e, float* __restrict__ dpos) {
  __shared__ __attribute__((aligned(16))) float joined[16][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.x;
  for (int base = 0; base < e; base += 512) {
    const int c = base + lane * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < e) {
      for (int b = wave; b < seqs; b += 64) {  // four sequences in flight
        V8<T> v[4];
        bool ok[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int s = min(b + 16 * j, seqs - 1), a = starts[s];
          ok[j] = b + 16 * j < seqs && t < starts[s + 1] - a;
          v[j] = v8_load_clamped<T>(dy, (size_t)(a + t) * e + c, ok[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f[8];
          v8_unpack(v8_mask(v[j], ok[j]), f);
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] += f[k];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) joined[wave][lane * 8 + k] = acc[k];
    __syncthreads();
    for (int k = threadIdx.x; k < 512 && base + k < e; k += 1024) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 16; ++w) s += joined[w][k];
      dpos[(size_t)t * e + base + k] = s;
    }
    __syncthreads();
  }
}

// forward: a workgroup takes one item of the layout's work list (or, without a layout, 32 consecutive rows); 8 columns a thread
template <typename T>
__global__ __launch_bounds__(256) void embed_packed_fwd_kernel(const long long* __restrict__ ids, const float* __restrict__ table, const float* __restrict__ pos,
                                                               const int* __restrict__ plan, int seqs, int block, int rows, int vocab, int positions, int e,
                                                               float scale, T* __restrict__ out) {
  int start = 0, len = rows, first = blockIdx.x * block, seq = 0;
  if (plan != nullptr) {
    const int* list = plan + ((seqs + 2) & ~1);
    seq = list[2 * blockIdx.x];
    if (seq < -1) return;
    first = list[2 * blockIdx.x + 1] * block;
    start = plan[seq >= 0 ? seq : seqs];
    len = (seq >= 0 ? plan[seq + 1] : rows) - start;
  }
  const int groups = e / 8, count = min(block, len - first);
  for (int i = threadIdx.x; i < count * groups; i += 256) {
    const int r = i / groups, c = (i - r * groups) * 8, place = first + r;
    const size_t row = (size_t)start + place;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (seq >= 0) {
      const long long t = ids[row];
      if (t >= 0 && t < vocab && (pos == nullptr || place < positions)) {
        v8_unpack(v8_load<float>(table + (size_t)t * e + c), f);
        if (pos != nullptr) {
          float g[8];
          v8_unpack(v8_load<float>(pos + (size_t)place * e + c), g);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = fmaf(f[k], scale, g[k]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] *= scale;
        }
      } else {  // a token outside the table, or a place without a position: said with NaN instead of a read out of bounds
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = __builtin_nanf("");
      }
    }
    V8<T> o;
    v8_pack(f, o);
    v8_store<T>(out + row * e + c, o);
  }
}

int sort_passes(int vocab) {
  int bits = 1;
  while (bits < 32 && ((unsigned)vocab >> bits)) ++bits;  // keys are 0 .. vocab
  return (bits + 7) / 8;
}
long long sort_blocks(long long n) { return (n + kItems - 1) / kItems; }

}  // namespace

// int32 scratch: two key and two row arrays, the digit counts
extern "C" long long cvh_embed_sort_elems(int rows) {
  if (rows <= 0) return -2;
  return 4ll * rows + sort_blocks(rows) * 256;
}
extern "C" long long cvh_embed_pieces_elems(int rows, int e) {
  if (rows <= 0 || e <= 0) return -2;
  return ((long long)rows + kChunk - 1) / kChunk * 2 * e;
}
extern "C" int cvh_embed_packed_fwd(int dtype, const long long* ids, const float* table, const float* pos, const int* plan, int seqs, int block, int places,
                                    int rows, int vocab, int positions, int e, float scale, void* out, void* stream) {
  if (dtype != CVH_DT_F32 && dtype != CVH_DT_BF16) return -1;
  if (ids == nullptr || table == nullptr || out == nullptr || rows <= 0 || vocab <= 0 || e <= 0 || e % 8 || (pos != nullptr && (plan == nullptr || positions <= 0))) return -2;
  if (plan != nullptr && (seqs <= 0 || (block != 32 && block != 128) || places != rows / block + seqs + 1)) return -2;
  if (plan == nullptr) {
    block = 32;
    places = (rows + block - 1) / block;
  }
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CVH_DT_BF16)
    hipLaunchKernelGGL(embed_packed_fwd_kernel<bf16_t>, dim3(places), dim3(256), 0, st, ids, table, pos, plan, seqs, block, rows, vocab, positions, e, scale, (bf16_t*)out);
  else
    hipLaunchKernelGGL(embed_packed_fwd_kernel<float>, dim3(places), dim3(256), 0, st, ids, table, pos, plan, seqs, block, rows, vocab, positions, e, scale, (float*)out);
  CVH_CHECK_LAUNCH();
  return 0;
}

template <typename T> static void embed_bwd(const T* dy, const unsigned* keys, const int* order, int rows, int vocab, int e, float scale, float* part, float* dtable, hipStream_t st) {
  const int chunks = (rows + kChunk - 1) / kChunk;
  if (rows > kChunk) hipLaunchKernelGGL(embed_pieces_kernel<T>, dim3((chunks + 3) / 4), dim3(256), 0, st, dy, keys, order, rows, vocab, e, part);
  int group = 4;
  while (group < 64 && group * 8 < e) group *= 2;
  hipLaunchKernelGGL(embed_rows_kernel<T>, dim3((vocab + kTableRows - 1) / kTableRows), dim3(256), 0, st, dy, keys, order, rows, vocab, e, scale, part, dtable, group);
}

extern "C" int cvh_embed_packed_bwd(int dtype, const long long* ids, const void* dout, const int* plan, int seqs, int rows, int vocab, int e, long long padding_idx,
                                    float scale, float* dtable, int positions, float* dpos, int* sort, float* pieces, void* stream) {
  if (dtype != CVH_DT_F32 && dtype != CVH_DT_BF16) return -1;
  if (dout == nullptr || rows <= 0 || e <= 0 || e % 8 || (dpos != nullptr && (plan == nullptr || positions <= 0)) || (plan != nullptr && seqs <= 0)) return -2;
  if (dtable != nullptr && (ids == nullptr || sort == nullptr || pieces == nullptr || vocab <= 0 || vocab >= 0x7fffffff - kTableRows)) return -2;
  hipStream_t st = (hipStream_t)stream;
  if (dtable != nullptr) {
    const int blocks = (int)sort_blocks(rows), passes = sort_passes(vocab);
    unsigned* keys[2] = {(unsigned*)sort, (unsigned*)sort + rows};
    int* order[2] = {sort + 2ll * rows, sort + 3ll * rows};
    int* count = sort + 4ll * rows;
    SortIn s = {ids, plan, nullptr, nullptr, padding_idx, rows, seqs, vocab, 0};
    for (int p = 0; p < passes; ++p) {
      s.shift = 8 * p;
      if (blocks > 1) hipLaunchKernelGGL(sort_count_kernel, dim3(blocks), dim3(256), 0, st, s, count);
      hipLaunchKernelGGL(sort_scatter_kernel, dim3(blocks), dim3(256), 0, st, s, count, keys[p & 1], order[p & 1]);
      s.keys = keys[p & 1];
      s.rows = order[p & 1];
    }
    if (dtype == CVH_DT_BF16) embed_bwd<bf16_t>((const bf16_t*)dout, s.keys, s.rows, rows, vocab, e, scale, pieces, dtable, st);
    else embed_bwd<float>((const float*)dout, s.keys, s.rows, rows, vocab, e, scale, pieces, dtable, st);
  }
  if (dpos != nullptr) {
    if (dtype == CVH_DT_BF16) hipLaunchKernelGGL(embed_pos_kernel<bf16_t>, dim3(positions), dim3(1024), 0, st, (const bf16_t*)dout, plan, seqs, e, dpos);
    else hipLaunchKernelGGL(embed_pos_kernel<float>, dim3(positions), dim3(1024), 0, st, (const float*)dout, plan, seqs, e, dpos);
  }
  CVH_CHECK_LAUNCH();
  return 0;
}
