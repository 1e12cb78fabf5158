// Token embedding on packed rows and its gradient by sorted tokens.
//
//   y_r = scale * table[id_r] + pos[r - cu[seq(r)]]
//   dtable[v] = scale * sum over { r : id_r = v } of dy_r, in the order of r;     dpos[t] = sum over the sequences b longer than t of dy[cu_b + t]
//
// The gradient of the table is dense float32.  Scattering with float atomics makes its sums depend on the order in which they retire and needs
// the table zeroed first; here the rows are sorted by token (stable radix sort, 8 bits a pass), every row of the table is then written exactly
// once, as the sum of its run in a fixed order: bit-reproducible.  What bounds it: the write of the whole table (49408 x 512: 101 MB) next to
// one read of dy (two with positions).  The sorted rows are summed in equal chunks, not token by token: frequent tokens (the start mark of every
// caption, the first words of a vocabulary in order of frequency) would otherwise leave their long runs to a few waves.
// Measured (26.7 k caption tokens, 49408 x 512, bf16 rows, positions): forward 14 us, two sort passes 12 us each, the gradient kernel 24 us for 101 MB of
// table and 55 MB of dy (positions read it again), joins 6 us.
#include "common.hpp"
#include "cvnets_hip.h"

namespace {

constexpr int kItems = 1024;   // rows a sort workgroup takes: 4 waves x 4 rounds x 64 lanes
constexpr int kChunk = 32;     // sorted rows that are summed by one group of lanes
constexpr int kTableRows = 32;  // rows of the table a workgroup writes
constexpr int kMostRows = 0x7fffffff - 4096, kMostBlocks = 1 << 24;  // (a grid has fewer than 2^32 threads)
constexpr int kMostPositions = 1 << 22;
// A scatter workgroup reads the counts of all workgroups where there are at most so many, which costs less than the launch that scans them; beyond, that
// would grow with the square of the rows (forward and gradient of 64, 128, 256, 1024, 4096 k rows x 32, a token each of 50000: 52 / 54, 69 / 67, 96 / 82,
// 332 / 222, 2286 / 642 us).
constexpr int kAllCounts = 96;

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

// The counts turned into places, in place: of each digit, the rows in earlier workgroups; behind the last workgroup's line: the rows of each digit in all.  A
// workgroup takes 32 digits, 32 lanes a line; each of its 32 groups of lanes a run of consecutive workgroups' counts.
__global__ __launch_bounds__(1024) void sort_scan_kernel(int* __restrict__ count, int blocks) {
  __shared__ int sum[32][32];
  const int digit = threadIdx.x & 31, group = threadIdx.x >> 5;
  int* const at = count + blockIdx.x * 32 + digit;
  const int per = (blocks + 31) / 32, b0 = min(group * per, blocks), b1 = min(b0 + per, blocks);
  int s = 0;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) s += at[(size_t)b * 256];
  sum[group][digit] = s;
  __syncthreads();
  int run = 0, total = 0;
  for (int g = 0; g < 32; ++g) {
    if (g == group) run = total;
    total += sum[g][digit];
  }
  for (int b = b0; b < b1; b += 8) {
    int v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at[(size_t)min(b + j, b1 - 1) * 256];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (b + j < b1) at[(size_t)(b + j) * 256] = run;
      run += v[j];
    }
  }
  if (group == 0) at[(size_t)blocks * 256] = total;
}

// stable scatter of one pass.  A wave's rows are consecutive; a lane's place = rows of smaller digits + of this digit in earlier workgroups, waves
// and rounds + in lower lanes of its round (8 ballots find the lanes with the same digit).
// count: the workgroups' counts, or (scanned) what sort_scan_kernel made of them.
__global__ __launch_bounds__(256) void sort_scatter_kernel(SortIn s, const int* __restrict__ count, int scanned, unsigned* __restrict__ keys_out, int* __restrict__ rows_out) {
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
  } else if (scanned) {
    before = count[(size_t)blockIdx.x * 256 + tid];
    total = count[(size_t)gridDim.x * 256 + tid];
  } else {
    for (int b0 = 0; b0 < (int)gridDim.x; b0 += 16) {
      int v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = count[min(b0 + j, (int)gridDim.x - 1) * 256 + tid];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int b = b0 + j, n = b < (int)gridDim.x ? v[j] : 0;
        before += b < (int)blockIdx.x ? n : 0;
        total += n;
      }
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

// ---- sums -------------------------------------------------------------------------------------------------------------------------------
// Chunk c of the sorted rows is [kChunk c, kChunk c + kChunk).  A run of one token that begins and ends in a chunk is written to the table at once;
// of a run that crosses borders every chunk leaves a piece: part[c][1] of the run that begins in chunk c and goes on, part[c][0] of the one
// that came in.  `G` lanes (8 columns each) share a chunk, so narrow tables keep whole waves busy.
__device__ __forceinline__ void put8(float* p, const float* acc, float scale) {
  *reinterpret_cast<float4*>(p) = make_float4(acc[0] * scale, acc[1] * scale, acc[2] * scale, acc[3] * scale);
  *reinterpret_cast<float4*>(p + 4) = make_float4(acc[4] * scale, acc[5] * scale, acc[6] * scale, acc[7] * scale);
}
__device__ __forceinline__ void add8(float* acc, const float* f) {
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] += f[k];
}

struct Grad {
  const unsigned* keys;  // sorted tokens
  const int* order;      // and their rows
  const int* starts;     // boundaries of the sequences
  float *dtable, *part, *dpos, *pos_part;
  int n, vocab, e, group, chunk_blocks, pos_blocks, seqs, pos_split;
  float scale;
};

template <typename T> __device__ __forceinline__ void chunk_rows(const Grad& g, const T* __restrict__ dy, int block) {
  const int G = g.group, chunk = block * (256 / G) + threadIdx.x / G, sl = threadIdx.x % G;
  const int a = chunk * kChunk, b = min(a + kChunk, g.n);
  if (a >= g.n) return;
  const bool came_in = a > 0 && g.keys[a - 1] == g.keys[a], goes_on = b < g.n && g.keys[b] == g.keys[b - 1];
  for (int c = sl * 8; c < g.e; c += G * 8) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    bool inside = !came_in;  // the run began in this chunk
    for (int i = a; i < b; i += 8) {  // eight rows in flight; keys and order are padded to whole chunks
      const uint4 k0 = *reinterpret_cast<const uint4*>(g.keys + i), k1 = *reinterpret_cast<const uint4*>(g.keys + i + 4);
      const int4 o0 = *reinterpret_cast<const int4*>(g.order + i), o1 = *reinterpret_cast<const int4*>(g.order + i + 4);
      const unsigned key[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
      const int row[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
      V8<T> v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v8_load_clamped<T>(dy, (size_t)row[j] * g.e + c, i + j < b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i + j >= b) break;
        float f[8];
        v8_unpack(v[j], f);
        add8(acc, f);
        const bool last = i + j + 1 == b;
        const unsigned next = last ? 0xffffffffu : j < 7 ? key[(j + 1) & 7] : g.keys[i + 8];
        if (last ? true : next != key[j]) {  // the run ends here, or the chunk does
          if (key[j] < (unsigned)g.vocab) {
            if (!inside) put8(g.part + ((size_t)chunk * 2) * g.e + c, acc, 1.f);
            else if (last && goes_on) put8(g.part + ((size_t)chunk * 2 + 1) * g.e + c, acc, 1.f);
            else put8(g.dtable + (size_t)key[j] * g.e + c, acc, g.scale);
          }
          inside = true;
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = 0.f;
        }
      }
    }
  }
}

// rows of the table that no token names: zeros
__device__ __forceinline__ void empty_rows(const Grad& g, int block) {
  __shared__ int bound[kTableRows + 1];
  __shared__ int range[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int v0 = block * kTableRows, rows = min(kTableRows, g.vocab - v0);
  if (wave < 2) {
    const int at = lower_bound_wave(g.keys, 0, g.n, (unsigned)(wave ? v0 + rows : v0), lane);
    if (lane == 0) range[wave] = at;
  }
  __syncthreads();
  if (tid <= rows) bound[tid] = lower_bound_lane(g.keys, range[0], range[1], (unsigned)(v0 + tid));
  __syncthreads();
  const int per = g.e / 4;
  float4* const out = reinterpret_cast<float4*>(g.dtable + (size_t)v0 * g.e);
  for (int i = tid; i < rows * per; i += 256) {
    const int r = i / per;
    if (bound[r] == bound[r + 1]) out[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// position t, one part of the sequences: the rows at that place; a wave takes 16 sequences at a time, eight rows in flight
template <typename T> __device__ __forceinline__ void pos_rows(const Grad& g, const T* __restrict__ dy, int block) {
  __shared__ __attribute__((aligned(16))) float joined[4][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = block / g.pos_split, part = block % g.pos_split;
  const int per = ((g.seqs + g.pos_split - 1) / g.pos_split + 63) & ~63, s0 = part * per, s1 = min(s0 + per, g.seqs);
  for (int base = 0; base < g.e; base += 512) {
    const int c = base + lane * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = s0 + wave * 16; s < s1; s += 64) {
      const int q = min(s + (lane & 15), g.seqs - 1), first = g.starts[q], row = first + t;
      unsigned m = (unsigned)(__ballot(s + (lane & 15) < s1 && t < g.starts[q + 1] - first) & 0xffffu);
      while (m) {
        V8<T> v[8];
        unsigned have = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int w = m ? __ffs(m) - 1 : 0;
          have |= (m ? 1u : 0u) << j;
          m &= m - 1;
          v[j] = v8_load_clamped<T>(dy, (size_t)__shfl(row, w, 64) * g.e + c, ((have >> j) & 1u) && c < g.e);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float f[8];
          v8_unpack(v8_mask(v[j], (have >> j) & 1u), f);
          add8(acc, f);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) joined[wave][lane * 8 + k] = acc[k];
    __syncthreads();
    float* const out = g.pos_split > 1 ? g.pos_part + ((size_t)part * (g.pos_blocks / g.pos_split) + t) * g.e : g.dpos + (size_t)t * g.e;
    for (int k = threadIdx.x; k < 512 && base + k < g.e; k += 256) out[base + k] = (joined[0][k] + joined[1][k]) + (joined[2][k] + joined[3][k]);
    __syncthreads();
  }
}

// the three kinds of workgroups of the backward pass: chunks (the longest ones) first, zeros last
template <typename T> __global__ __launch_bounds__(256) void embed_grad_kernel(Grad g, const T* __restrict__ dy) {
  const int block = blockIdx.x;
  if (block < g.chunk_blocks) chunk_rows<T>(g, dy, block);
  else if (block < g.chunk_blocks + g.pos_blocks) pos_rows<T>(g, dy, block - g.chunk_blocks);
  else empty_rows(g, block - g.chunk_blocks - g.pos_blocks);
}

// runs that cross chunks: the workgroup of the chunk that such a run begins in adds up its pieces, 256 / G of them side by side; and the parts of
// the positions' sums
__global__ __launch_bounds__(256) void embed_join_kernel(Grad g, int chunks) {
  __shared__ __attribute__((aligned(16))) float joined[2048];
  __shared__ int run_end;
  const int tid = threadIdx.x, G = g.group, per = 256 / G, sub = tid / G, sl = tid % G, item = blockIdx.y * gridDim.x + blockIdx.x;
  if (item >= chunks) {
    const int t = item - chunks, positions = g.pos_blocks / g.pos_split;
    if (g.pos_split == 1 || t >= positions) return;  // (the last line of the grid)
    for (int c = tid; c < g.e; c += 256) {
      float s = 0.f;
#pragma unroll 8
      for (int q = 0; q < g.pos_split; ++q) s += g.pos_part[((size_t)q * positions + t) * g.e + c];
      g.dpos[(size_t)t * g.e + c] = s;
    }
    return;
  }
  const int chunk = item, a = chunk * kChunk, b = a + kChunk;
  if (b >= g.n) return;
  const unsigned v = g.keys[b - 1];
  if (v >= (unsigned)g.vocab || g.keys[b] != v || (a > 0 && g.keys[a - 1] == v)) return;  // does not go on, or came in (the same for all threads)
  if (tid < 64) {
    const int at = lower_bound_wave(g.keys, b, g.n, v + 1, tid);
    if (tid == 0) run_end = at;
  }
  __syncthreads();
  const int last = (run_end - 1) / kChunk;
  for (int base = 0; base < g.e; base += G * 8) {
    const int c = base + sl * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < g.e) {
#pragma unroll 8
      for (int k = chunk + sub; k <= last; k += per) {
        const float* p = g.part + ((size_t)k * 2 + (k == chunk ? 1 : 0)) * g.e + c;
        const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
        const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        add8(acc, f);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) joined[tid * 8 + k] = acc[k];
    __syncthreads();
    for (int k = tid; k < G * 8 && base + k < g.e; k += 256) {
      float s = 0.f;
      for (int q = 0; q < per; ++q) s += joined[q * G * 8 + k];
      g.dtable[(size_t)v * g.e + base + k] = s * g.scale;
    }
    __syncthreads();
  }
}

// forward: a workgroup takes `share` rows of one item of the layout's work list (or, without a layout, of 32 consecutive rows); 8 columns a thread
template <typename T>
__global__ __launch_bounds__(256) void embed_packed_fwd_kernel(const long long* __restrict__ ids, const float* __restrict__ table, const float* __restrict__ pos,
                                                               const int* __restrict__ plan, int seqs, int block, int share, int rows, int vocab, int positions,
                                                               int e, float scale, T* __restrict__ out) {
  int start = 0, len = rows, first = blockIdx.x * block, seq = 0;
  if (plan != nullptr) {
    const int* list = plan + ((seqs + 2) & ~1);
    seq = list[2 * blockIdx.x];
    if (seq < -1) return;
    first = list[2 * blockIdx.x + 1] * block;
    start = plan[seq >= 0 ? seq : seqs];
    len = (seq >= 0 ? plan[seq + 1] : rows) - start;
  }
  first += blockIdx.y * share;
  const int groups = e / 8, count = min(share, len - first);
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
long long padded(long long n) { return (n + kChunk - 1) / kChunk * kChunk; }
// 64 sequences a workgroup, while that is at most 16 parts; one part where the positions alone are more workgroups than the card takes at a time
int pos_split(int seqs, int positions) { return seqs <= 64 || positions > 1 << 18 ? 1 : seqs >= 1024 ? 16 : (seqs + 63) / 64; }

}  // namespace

// int32 scratch: two key and two row arrays (in whole chunks), the digit counts
extern "C" long long cvh_embed_sort_elems(int rows) {
  if (rows <= 0 || rows > kMostRows) return -2;
  return 4 * padded(rows) + (sort_blocks(rows) + 1) * 256;
}
// float32 scratch: two pieces a chunk, the parts of the positions' sums
extern "C" long long cvh_embed_pieces_elems(int rows, int e, int positions, int seqs) {
  if (rows <= 0 || rows > kMostRows || e <= 0 || positions < 0 || positions > kMostPositions || seqs < 0) return -2;
  const int split = pos_split(seqs, positions);
  return (padded(rows) / kChunk * 2 + (split > 1 ? (long long)split * positions : 0)) * e;
}
extern "C" int cvh_embed_packed_fwd(int dtype, const long long* ids, const float* table, const float* pos, const int* plan, int seqs, int block, int places,
                                    int rows, int vocab, int positions, int e, float scale, void* out, void* stream) {
  if (dtype != CVH_DT_F32 && dtype != CVH_DT_BF16) return -1;
  if (ids == nullptr || table == nullptr || out == nullptr || rows <= 0 || rows > kMostRows || vocab <= 0 || e <= 0 || e % 8 || (pos != nullptr && (plan == nullptr || positions <= 0 || positions > kMostPositions))) return -2;
  if (plan != nullptr && (seqs <= 0 || (block != 32 && block != 128) || places != (long long)rows / block + seqs + 1)) return -2;
  if (plan == nullptr) {
    block = rows < 1 << 28 ? 32 : 128;
    places = (rows + block - 1) / block;
  }
  if (places >= kMostBlocks) return -2;
  hipStream_t st = (hipStream_t)stream;
  int share = block;  // about 2048 pieces of 8 columns a workgroup: 25 k rows of 768 in 128-row items are 232 workgroups otherwise, fewer than CUs
  while (share > 8 && share * (e / 8) > 2048) share /= 2;
  const dim3 grid(places, block / share);
  if (dtype == CVH_DT_BF16)
    hipLaunchKernelGGL(embed_packed_fwd_kernel<bf16_t>, grid, dim3(256), 0, st, ids, table, pos, plan, seqs, block, share, rows, vocab, positions, e, scale, (bf16_t*)out);
  else
    hipLaunchKernelGGL(embed_packed_fwd_kernel<float>, grid, dim3(256), 0, st, ids, table, pos, plan, seqs, block, share, rows, vocab, positions, e, scale, (float*)out);
  CVH_CHECK_LAUNCH();
  return 0;
}

extern "C" int cvh_embed_packed_bwd(int dtype, const long long* ids, const void* dout, const int* plan, int seqs, int rows, int vocab, int e, long long padding_idx,
                                    float scale, float* dtable, int positions, float* dpos, int* sort, float* pieces, void* stream) {
  if (dtype != CVH_DT_F32 && dtype != CVH_DT_BF16) return -1;
  if (dout == nullptr || rows <= 0 || rows > kMostRows || e <= 0 || e % 8 || (dpos != nullptr && (plan == nullptr || positions <= 0 || positions > kMostPositions || pieces == nullptr)) || (plan != nullptr && seqs <= 0)) return -2;
  if (dtable != nullptr && (ids == nullptr || sort == nullptr || pieces == nullptr || vocab <= 0 || vocab / kTableRows >= kMostBlocks / 2)) return -2;
  hipStream_t st = (hipStream_t)stream;
  Grad g = {};
  g.n = rows; g.vocab = vocab; g.e = e; g.scale = scale; g.starts = plan; g.seqs = seqs;
  g.dtable = dtable; g.part = pieces; g.dpos = dpos;
  g.group = 4;
  while (g.group < 64 && g.group * 8 < e) g.group *= 2;
  int zero_blocks = 0, chunks = 0;
  if (dtable != nullptr) {
    const int blocks = (int)sort_blocks(rows), passes = sort_passes(vocab);
    const long long size = padded(rows);
    unsigned* keys[2] = {(unsigned*)sort, (unsigned*)sort + size};
    int* order[2] = {sort + 2 * size, sort + 3 * size};
    int* count = sort + 4 * size;
    SortIn s = {ids, plan, nullptr, nullptr, padding_idx, rows, seqs, vocab, 0};
    for (int p = 0; p < passes; ++p) {
      s.shift = 8 * p;
      if (blocks > 1) hipLaunchKernelGGL(sort_count_kernel, dim3(blocks), dim3(256), 0, st, s, count);
      const int scanned = blocks > kAllCounts;
      if (scanned) hipLaunchKernelGGL(sort_scan_kernel, dim3(8), dim3(1024), 0, st, count, blocks);
      hipLaunchKernelGGL(sort_scatter_kernel, dim3(blocks), dim3(256), 0, st, s, count, scanned, keys[p & 1], order[p & 1]);
      s.keys = keys[p & 1];
      s.rows = order[p & 1];
    }
    g.keys = s.keys;
    g.order = s.rows;
    chunks = (int)(size / kChunk);
    g.chunk_blocks = (chunks + 256 / g.group - 1) / (256 / g.group);
    zero_blocks = (vocab + kTableRows - 1) / kTableRows;
  }
  g.pos_split = 1;
  if (dpos != nullptr) {
    g.pos_split = pos_split(seqs, positions);
    g.pos_blocks = positions * g.pos_split;
    g.pos_part = pieces + (long long)padded(rows) / kChunk * 2 * e;
  }
  if ((long long)g.chunk_blocks + g.pos_blocks + zero_blocks >= kMostBlocks) return -2;
  const dim3 grid(g.chunk_blocks + g.pos_blocks + zero_blocks);
  if (grid.x == 0) return 0;
  if (dtype == CVH_DT_BF16) hipLaunchKernelGGL(embed_grad_kernel<bf16_t>, grid, dim3(256), 0, st, g, (const bf16_t*)dout);
  else hipLaunchKernelGGL(embed_grad_kernel<float>, grid, dim3(256), 0, st, g, (const float*)dout);
  const int joins = (chunks > 1 ? chunks : 0) + (g.pos_split > 1 ? positions : 0);
  constexpr int kLine = 1 << 22;  // (2^26 chunks of 2^31 rows: lines of a grid)
  if (joins > 0) hipLaunchKernelGGL(embed_join_kernel, dim3(joins < kLine ? joins : kLine, (joins + kLine - 1) / kLine), dim3(256), 0, st, g, chunks > 1 ? chunks : 0);
  CVH_CHECK_LAUNCH();
  return 0;
}
