// A token embedding's lookup, the gradient of its weight, and how often each
// token occurs (the diagonal of the input factor of its K-FAC block).
//
// lookup    out[i] = scale * W[id_i]
// gradient  dW[v] = scale * sum over {i : id_i = v} of gy[i]
//
// The gradient sorts the tokens first (stable, so that a row's sum always runs in
// the order of the positions: no atomics on values, the same bits every time) and
// then walks the sorted positions in chunks; a token whose positions pass the end of
// a chunk leaves partial sums, which a second launch adds up in order.  Rows of
// tokens that do not occur are cleared by blocks of the same launch.
//
// Bound: HBM.  A lookup reads the distinct rows and writes n rows; a gradient reads
// n rows and writes all rows of the weight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace kfac {
namespace {

// ------------------------------------------------------------------ tokens

struct Ids {
  const void* p;
  int wide;              // 64-bit
  int has_ignore;
  long long ignore;
  long long n;
  int vocab;
};

// What a lookup makes of a token: its row, kIgnored (zeros) or kOutside (no row of
// the weight: NaN).
constexpr int kIgnored = -1, kOutside = -2;
__device__ __forceinline__ int row_of(const Ids& s, long long i) {
  const long long id = s.wide ? static_cast<const long long*>(s.p)[i]
                              : static_cast<const int*>(s.p)[i];
  if (s.has_ignore && id == s.ignore) return kIgnored;
  return id >= 0 && id < s.vocab ? (int)id : kOutside;
}

// Its key in the sort: tokens without a row come last.
__device__ __forceinline__ int key_of(const Ids& s, long long i) {
  const int r = row_of(s, i);
  return r >= 0 ? r : s.vocab;
}

// ------------------------------------------------------------------ values

template <typename T> struct Num;
template <> struct Num<float> {
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Num<__half> {
  static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
};
template <> struct Num<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 x) {
    return __bfloat162float(x);
  }
  static __device__ __forceinline__ __nv_bfloat16 put(float x) {
    return __float2bfloat16_rn(x);
  }
};

// V values of type T that are read and written as one word.
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T x[V];
};

// ------------------------------------------------------------------ lookup

constexpr int kLookThreads = 256;
constexpr int kLookRows = 4;      // rows a thread has in flight

// `lanes` threads (a power of two) share a row; a block has kLookThreads / lanes
// rows at a time, kLookRows times.
template <typename T, int V>
__global__ void __launch_bounds__(kLookThreads)
embed_lookup_kernel(const T* __restrict__ weight, const Ids ids, int width,
                    float scale, T* __restrict__ out, int lanes) {
  using P = Pack<T, V>;
  const int per = kLookThreads / lanes;
  const int at = threadIdx.x & (lanes - 1), sub = threadIdx.x / lanes;
  const int words = width / V;
  const long long step = (long long)gridDim.x * per * kLookRows;
  for (long long i0 = (long long)blockIdx.x * per * kLookRows; i0 < ids.n;
       i0 += step) {
    int row[kLookRows];
#pragma unroll
    for (int u = 0; u < kLookRows; ++u) {
      const long long i = i0 + (long long)u * per + sub;
      row[u] = i < ids.n ? row_of(ids, i) : kIgnored;
    }
    for (int w = at; w < words; w += lanes) {
      P x[kLookRows];
#pragma unroll
      for (int u = 0; u < kLookRows; ++u)
        if (row[u] >= 0)
          x[u] = *reinterpret_cast<const P*>(weight + (long long)row[u] * width +
                                             (long long)w * V);
#pragma unroll
      for (int u = 0; u < kLookRows; ++u) {
        const long long i = i0 + (long long)u * per + sub;
        if (i >= ids.n) continue;
        const float none = row[u] == kIgnored ? 0.f : __int_as_float(0x7fc00000);
#pragma unroll
        for (int e = 0; e < V; ++e)
          x[u].x[e] = Num<T>::put(row[u] >= 0 ? scale * Num<T>::get(x[u].x[e])
                                              : none);
        *reinterpret_cast<P*>(out + i * width + (long long)w * V) = x[u];
      }
    }
  }
}

// -------------------------------------------------------------------- sort
// Least significant digit first, digits of up to 9 bits: two passes for a vocabulary
// of up to 2^18 - 1 (one key more than tokens: those without a row).  Keys stay in
// their order within a digit: a warp takes 32 x kSortItems consecutive keys, 32 at a
// time; lanes with the same digit find each other by a match, and the warp's own
// counters say how many came before.

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kDigitBits = 9;
constexpr int kBins = 1 << kDigitBits;
static_assert(kBins == kSortThreads, "a thread per bin");
constexpr int kOwnBases = 64;    // most tiles whose counts a block adds up itself

struct Digit {
  int shift, mask;
};

struct SortCounts {
  int warp[kSortWarps][kBins];   // keys of a warp with a digit, then of those before
  int base[kBins];               // where the tile's first key with a digit goes
  int part[kSortWarps];
};

// Place of each of the thread's keys among its warp's with the same digit, and the
// warp's counts.  `live`: keys there are (the others behind them).
template <int ITEMS>
__device__ __forceinline__ void rank_keys(SortCounts& s, const int (&key)[ITEMS],
                                          Digit d, int (&rank)[ITEMS]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = lane; b < kBins; b += 32) s.warp[warp][b] = 0;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int digit = (key[j] >> d.shift) & d.mask;
    const unsigned peers = __match_any_sync(0xffffffffu, digit);
    const int before = s.warp[warp][digit];
    __syncwarp();
    rank[j] = before + __popc(peers & ((1u << lane) - 1));
    if (lane == 31 - __clz(peers)) s.warp[warp][digit] = before + __popc(peers);
    __syncwarp();
  }
}

// Counts of the warps in front, and the tile's own count of the thread's digit.
__device__ __forceinline__ int count_before(SortCounts& s) {
  int run = 0;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) {
    const int c = s.warp[w][threadIdx.x];
    s.warp[w][threadIdx.x] = run;
    run += c;
  }
  return run;
}

// Sum of `x` over the threads in front of this one.
__device__ __forceinline__ int sum_before(SortCounts& s, int x) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) s.part[warp] = inc;
  __syncthreads();
  int front = 0;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) front += w < warp ? s.part[w] : 0;
  __syncthreads();
  return front + inc - x;
}

// All passes of up to kSortTile tokens by one block.
__global__ void __launch_bounds__(kSortThreads)
token_sort_tile_kernel(const Ids ids, int bits, int passes, int* keys_out,
                       int* perm_out) {
  extern __shared__ unsigned char sort_smem[];
  SortCounts& s = *reinterpret_cast<SortCounts*>(sort_smem);
  int* keys = reinterpret_cast<int*>(sort_smem + sizeof(SortCounts));
  unsigned short* perm = reinterpret_cast<unsigned short*>(keys + kSortTile);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = warp * 32 * kSortItems + lane;
  const int n = (int)ids.n;
  int key[kSortItems], pos[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    pos[j] = first + 32 * j;
    key[j] = pos[j] < n ? key_of(ids, pos[j]) : 0x7fffffff;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const Digit d = {pass * bits, (1 << bits) - 1};
    rank_keys(s, key, d, rank);
    __syncthreads();
    const int mine = count_before(s);
    s.base[threadIdx.x] = sum_before(s, mine);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const int digit = (key[j] >> d.shift) & d.mask;
      const int to = s.base[digit] + s.warp[warp][digit] + rank[j];
      keys[to] = key[j];
      perm[to] = (unsigned short)pos[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      key[j] = keys[first + 32 * j];
      pos[j] = perm[first + 32 * j];
    }
    __syncthreads();
  }
  // (a key behind the end is larger than any other in every digit)
#pragma unroll
  for (int j = 0; j < kSortItems; ++j)
    if (first + 32 * j < n) {
      keys_out[first + 32 * j] = key[j];
      perm_out[first + 32 * j] = pos[j];
    }
}

// Keys of a tile; those of the first pass come from the tokens themselves.
__device__ __forceinline__ int sort_key(const Ids& ids, const int* keys,
                                        long long i) {
  if (i >= ids.n) return 0x7fffffff;
  return keys == nullptr ? key_of(ids, i) : keys[i];
}

// Counts of a tile's digits: counts[tile][digit].
__global__ void __launch_bounds__(kSortThreads)
token_count_kernel(const Ids ids, const int* keys, Digit d, int* counts) {
  __shared__ int bins[kBins];
  bins[threadIdx.x] = 0;
  __syncthreads();
  const long long i0 = (long long)blockIdx.x * kSortTile + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const long long i = i0 + j * kSortThreads;
    if (i < ids.n)
      atomicAdd(&bins[(sort_key(ids, keys, i) >> d.shift) & d.mask], 1);
  }
  __syncthreads();
  counts[(long long)blockIdx.x * kBins + threadIdx.x] = bins[threadIdx.x];
}

// Of more than kOwnBases tiles: every tile's first place of a digit.
__global__ void __launch_bounds__(kSortThreads)
token_bases_kernel(int* counts, int tiles) {
  __shared__ SortCounts s;
  int* mine = counts + threadIdx.x;
  int total = 0;
#pragma unroll 16
  for (int t = 0; t < tiles; ++t) total += mine[(long long)t * kBins];
  int run = sum_before(s, total);
#pragma unroll 8
  for (int t = 0; t < tiles; ++t) {
    const int c = mine[(long long)t * kBins];
    mine[(long long)t * kBins] = run;
    run += c;
  }
}

__global__ void __launch_bounds__(kSortThreads)
token_scatter_kernel(const Ids ids, const int* keys, const int* perm, Digit d,
                     const int* counts, int tiles, int* keys_out,
                     int* perm_out) {
  __shared__ SortCounts s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long first =
      (long long)blockIdx.x * kSortTile + warp * 32 * kSortItems + lane;
  int key[kSortItems], pos[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const long long i = first + 32 * j;
    key[j] = sort_key(ids, keys, i);
    pos[j] = perm == nullptr || i >= ids.n ? (int)i : perm[i];
  }
  int base;
  if (tiles <= kOwnBases) {
    int total = 0, before = 0;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
      const int c = counts[t * kBins + threadIdx.x];
      total += c;
      before += t < (int)blockIdx.x ? c : 0;
    }
    base = sum_before(s, total) + before;
  } else {
    base = counts[(long long)blockIdx.x * kBins + threadIdx.x];
  }
  s.base[threadIdx.x] = base;
  rank_keys(s, key, d, rank);
  __syncthreads();
  count_before(s);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    if (first + 32 * j >= ids.n) continue;
    const int digit = (key[j] >> d.shift) & d.mask;
    const int to = s.base[digit] + s.warp[warp][digit] + rank[j];
    keys_out[to] = key[j];
    perm_out[to] = pos[j];
  }
}

// ---------------------------------------------------------------- gradient

constexpr int kGradThreads = 128;
constexpr int kGradAhead = 8;       // rows in flight
constexpr int kClearRows = 32;      // rows of a block that clears

struct Grad {
  const int* keys;       // sorted
  const int* perm;
  long long n;
  int vocab, width;
  int chunk;             // sorted positions of a chunk
  int lanes;             // threads of a chunk and slab of columns
  int slabs;
  long long chunks;
  long long chunk_blocks;
  long long pitch;       // floats of a partial row
  float* part;           // [chunk][2]: of the token from before, of the last one
  float scale;
  int add;               // onto the rows that are there
};

template <typename T, int V>
__device__ __forceinline__ void put_row(T* out, const float (&acc)[V], float scale,
                                        bool add) {
  using P = Pack<T, V>;
  P x;
  if (add) x = *reinterpret_cast<const P*>(out);
#pragma unroll
  for (int e = 0; e < V; ++e)
    x.x[e] = Num<T>::put(add ? fmaf(scale, acc[e], Num<T>::get(x.x[e]))
                             : scale * acc[e]);
  *reinterpret_cast<P*>(out) = x;
}

template <typename T, int V>
__global__ void __launch_bounds__(kGradThreads)
embed_grad_kernel(const Grad g, const T* __restrict__ gy, T* __restrict__ out) {
  using P = Pack<T, V>;
  if (blockIdx.x >= g.chunk_blocks) {
    // rows of tokens that do not occur
    __shared__ unsigned clear;
    const int r0 = (int)((blockIdx.x - g.chunk_blocks) * kClearRows);
    if (threadIdx.x < 32) {
      const int r = r0 + threadIdx.x;
      long long lo = 0, hi = g.n;
      while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (g.keys[mid] < r) lo = mid + 1; else hi = mid;
      }
      const bool there = lo < g.n && g.keys[lo] == r;
      const unsigned m = __ballot_sync(0xffffffffu, !there && r < g.vocab);
      if (threadIdx.x == 0) clear = m;
    }
    __syncthreads();
    unsigned rows = clear;
    P zero;
#pragma unroll
    for (int e = 0; e < V; ++e) zero.x[e] = Num<T>::put(0.f);
    const int words = g.width / V;
    while (rows != 0) {
      const int r = r0 + __ffs(rows) - 1;
      rows &= rows - 1;
      P* to = reinterpret_cast<P*>(out + (long long)r * g.width);
      for (int w = threadIdx.x; w < words; w += kGradThreads) to[w] = zero;
    }
    return;
  }
  const int per = kGradThreads / g.lanes;
  const long long item = (long long)blockIdx.x * per + threadIdx.x / g.lanes;
  const long long chunk = item / g.slabs;
  const int col =
      ((int)(item - chunk * g.slabs) * g.lanes + (threadIdx.x & (g.lanes - 1))) * V;
  if (chunk >= g.chunks || col >= g.width) return;
  const long long p0 = chunk * g.chunk, p1 = min(p0 + g.chunk, g.n);
  const int before = p0 > 0 ? g.keys[p0 - 1] : -1;
  const int behind = p1 < g.n ? g.keys[p1] : -1;
  int cur = g.keys[p0];
  bool head = cur == before;
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  auto leave = [&](bool tail) {
    if (head || tail) {
      float* to = g.part + (2 * chunk + (head ? 0 : 1)) * g.pitch + col;
#pragma unroll
      for (int e = 0; e < V; ++e) to[e] = acc[e];
    } else {
      put_row<T, V>(out + (long long)cur * g.width + col, acc, g.scale, g.add);
    }
  };
  for (long long p = p0; p < p1 && cur != g.vocab; p += kGradAhead) {
    int key[kGradAhead];
    P x[kGradAhead];
#pragma unroll
    for (int u = 0; u < kGradAhead; ++u) {
      key[u] = p + u < p1 ? g.keys[p + u] : g.vocab;
      if (key[u] != g.vocab)
        x[u] = *reinterpret_cast<const P*>(
            gy + (long long)g.perm[p + u] * g.width + col);
    }
#pragma unroll
    for (int u = 0; u < kGradAhead; ++u) {
      if (p + u >= p1) break;
      if (key[u] != cur) {
        leave(false);
        cur = key[u];
        head = false;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
        if (cur == g.vocab) break;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += Num<T>::get(x[u].x[e]);
    }
  }
  if (cur != g.vocab) leave(cur == behind);
}

// Tokens whose positions lie in several chunks: the sum of their parts, a quarter of
// the chunks by each quarter of the block.
constexpr int kJoinCols = 128;
template <typename T>
__global__ void __launch_bounds__(4 * kJoinCols)
embed_join_kernel(const Grad g, T* __restrict__ out, int slabs) {
  __shared__ float sums[3][kJoinCols];
  __shared__ long long end;
  const long long chunk = blockIdx.x / slabs;
  const long long p0 = chunk * g.chunk, p1 = p0 + g.chunk;
  // the token that begins in this chunk and goes on behind it, if there is one
  if (p1 >= g.n) return;
  const int key = g.keys[p1];
  if (key == g.vocab || g.keys[p1 - 1] != key ||
      (p0 > 0 && g.keys[p0 - 1] == key))
    return;
  if (threadIdx.x == 0) {
    long long lo = p1 + 1, hi = g.n;     // first position behind the token's
    while (lo < hi) {
      const long long mid = (lo + hi) >> 1;
      if (g.keys[mid] <= key) lo = mid + 1; else hi = mid;
    }
    end = (lo - 1) / g.chunk + 1;        // first chunk without it
  }
  __syncthreads();
  const int quarter = threadIdx.x / kJoinCols;
  const int col = (int)(blockIdx.x - chunk * slabs) * kJoinCols +
                  (threadIdx.x & (kJoinCols - 1));
  const long long many = end - chunk;    // parts: this chunk's, then the others'
  const long long each = (many + 3) / 4;
  const long long c0 = chunk + quarter * each;
  const long long c1 = min(c0 + each, end);
  float sum = 0.f;
  if (col < g.width) {
#pragma unroll 8
    for (long long c = c0; c < c1; ++c)
      sum += g.part[(2 * c + (c == chunk ? 1 : 0)) * g.pitch + col];
  }
  if (quarter > 0) sums[quarter - 1][threadIdx.x & (kJoinCols - 1)] = sum;
  __syncthreads();
  if (quarter > 0 || col >= g.width) return;
  const float acc[1] = {sum + sums[0][threadIdx.x] + sums[1][threadIdx.x] +
                        sums[2][threadIdx.x]};
  put_row<T, 1>(out + (long long)key * g.width + col, acc, g.scale, g.add);
}

// ------------------------------------------------------------------ counts

__global__ void __launch_bounds__(256)
token_histogram_kernel(const Ids ids, int* counts) {
  const long long step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < ids.n; i += step) {
    const int r = row_of(ids, i);
    if (r >= 0) atomicAdd(&counts[r], 1);
  }
}

// out = alpha * counts + beta * out, and their mean the same way.  One block adds up
// the mean (its sum of whole numbers is exact).
__global__ void __launch_bounds__(256)
token_counts_kernel(const int* counts, int vocab, float alpha, float beta, float* out,
                    float* mean) {
  __shared__ long long part[8];
  if (blockIdx.x == gridDim.x - 1) {
    if (mean == nullptr) return;
    long long sum = 0;
    for (int v = threadIdx.x; v < vocab; v += 256) sum += counts[v];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) sum += part[w];
      const float m = (float)((double)alpha * (double)sum / (double)vocab);
      *mean = beta == 0.f ? m : m + beta * *mean;
    }
    return;
  }
  const long long v = (long long)blockIdx.x * 256 + threadIdx.x;
  if (v >= vocab) return;
  const float a = alpha * (float)counts[v];
  out[v] = beta == 0.f ? a : fmaf(beta, out[v], a);
}

// --------------------------------------------------------------- host side

long long parts_of(long long a, long long b) { return (a + b - 1) / b; }

size_t type_size(int dtype) { return dtype == KFAC_WIRE_F32 ? 4 : 2; }

// Bytes of the widest word that rows of `width` values at these addresses can be
// read in.
int word_bytes(const void* a, const void* b, int width, int dtype) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) |
                        reinterpret_cast<uintptr_t>(b) |
                        ((uintptr_t)width * type_size(dtype)) | 16;
  return (int)(all & (~all + 1));
}

int check_ids(const char* what, const void* ids, int id_bytes, int64_t n,
              int64_t vocab) {
  KFAC_REQUIRE(id_bytes == 4 || id_bytes == 8,
               "%s: tokens of %d bytes (4 or 8 are supported)", what, id_bytes);
  KFAC_REQUIRE(n >= 0 && n < (1LL << 31) - kSortTile, "%s: %lld tokens", what,
               (long long)n);
  KFAC_REQUIRE(vocab >= 1 && vocab < (1LL << 31) - 1,
               "%s: a vocabulary of %lld tokens", what, (long long)vocab);
  KFAC_REQUIRE(n == 0 || ids != nullptr, "%s: null pointer", what);
  return KFAC_OK;
}

int check_rows(const char* what, int dtype, int width) {
  KFAC_REQUIRE(dtype == KFAC_WIRE_F32 || dtype == KFAC_WIRE_F16 ||
                   dtype == KFAC_WIRE_BF16,
               "%s: unknown element type %d", what, dtype);
  KFAC_REQUIRE(width >= 1, "%s: rows of %d values", what, width);
  return KFAC_OK;
}

Ids make_ids(const void* ids, int id_bytes, int64_t n, int64_t vocab,
             int has_ignore, int64_t ignore) {
  Ids s;
  s.p = ids;
  s.wide = id_bytes == 8;
  s.has_ignore = has_ignore;
  s.ignore = ignore;
  s.n = n;
  s.vocab = (int)vocab;
  return s;
}

template <typename T, int V>
int look_up(const void* weight, const Ids& ids, int width, float scale, void* out,
            cudaStream_t st) {
  int lanes = 1;
  while (lanes < kLookThreads && lanes * V < width) lanes *= 2;
  const long long rows = (long long)(kLookThreads / lanes) * kLookRows;
  const long long blocks = (ids.n + rows - 1) / rows;
  embed_lookup_kernel<T, V>
      <<<(unsigned)std::min<long long>(blocks, 1 << 20), kLookThreads, 0, st>>>(
          static_cast<const T*>(weight), ids, width, scale, static_cast<T*>(out),
          lanes);
  KFAC_LAUNCH_CHECK("embed_lookup_kernel");
  return KFAC_OK;
}

template <typename T>
int look_up_by(int word, const void* weight, const Ids& ids, int width, float scale,
               void* out, cudaStream_t st) {
  constexpr int S = (int)sizeof(T);
  switch (word) {
    case 16: return look_up<T, 16 / S>(weight, ids, width, scale, out, st);
    case 8: return look_up<T, 8 / S>(weight, ids, width, scale, out, st);
    case 4: return look_up<T, 4 / S>(weight, ids, width, scale, out, st);
    default: return look_up<T, 1>(weight, ids, width, scale, out, st);
  }
}

struct SortPlan {
  int bits, passes;
  long long tiles;
  size_t keys, counts;      // bytes of a spare key (and perm) array, of the counts
};

SortPlan plan_sort(int64_t n, int64_t vocab) {
  SortPlan p;
  int need = 1;
  while (need < 31 && (vocab >> need) != 0) ++need;      // keys 0 .. vocab
  p.passes = (need + kDigitBits - 1) / kDigitBits;
  p.bits = (need + p.passes - 1) / p.passes;
  p.tiles = (n + kSortTile - 1) / kSortTile;
  p.keys = p.tiles > 1 ? ((size_t)n * 4 + 255) & ~(size_t)255 : 0;
  p.counts = p.tiles > 1 ? (size_t)p.tiles * kBins * sizeof(int) : 0;
  return p;
}

// Chunks of the sorted positions: long enough that partial rows are few, short
// enough that there are blocks for every SM.
struct GradPlan {
  int lanes, slabs, chunk;
  long long chunks;
  long long pitch;
};

GradPlan plan_grad(int64_t n, int width, int v) {
  GradPlan p;
  p.lanes = 1;
  while (p.lanes < kGradThreads && p.lanes * v < width) p.lanes *= 2;
  p.slabs = (width + p.lanes * v - 1) / (p.lanes * v);
  p.chunk = 8;
  const long long per = kGradThreads / p.lanes;
  while (p.chunk < 64 &&
         parts_of(parts_of(n, p.chunk) * p.slabs, per) > 16 * 148)
    p.chunk *= 2;
  p.chunks = parts_of(n, p.chunk);
  p.pitch = ((long long)width + 3) & ~3LL;
  return p;
}

template <typename T, int V>
int run_grad(Grad g, const void* gy, void* out, cudaStream_t st) {
  const GradPlan p = plan_grad(g.n, g.width, V);
  g.chunk = p.chunk;
  g.lanes = p.lanes;
  g.slabs = p.slabs;
  g.chunks = p.chunks;
  g.pitch = p.pitch;
  g.chunk_blocks = parts_of(p.chunks * p.slabs, kGradThreads / p.lanes);
  const long long clear = g.add ? 0 : parts_of(g.vocab, kClearRows);
  const long long blocks = g.chunk_blocks + clear;
  KFAC_REQUIRE(blocks < (1LL << 31), "embedding_grad: too many blocks");
  if (blocks == 0) return KFAC_OK;
  embed_grad_kernel<T, V><<<(unsigned)blocks, kGradThreads, 0, st>>>(
      g, static_cast<const T*>(gy), static_cast<T*>(out));
  KFAC_LAUNCH_CHECK("embed_grad_kernel");
  if (p.chunks > 1) {
    const int slabs = ceil_div(g.width, kJoinCols);
    KFAC_REQUIRE(p.chunks * slabs < (1LL << 31), "embedding_grad: too many blocks");
    embed_join_kernel<T><<<(unsigned)(p.chunks * slabs), 4 * kJoinCols, 0, st>>>(
        g, static_cast<T*>(out), slabs);
    KFAC_LAUNCH_CHECK("embed_join_kernel");
  }
  return KFAC_OK;
}

template <typename T>
int run_grad_by(int word, const Grad& g, const void* gy, void* out,
                cudaStream_t st) {
  constexpr int S = (int)sizeof(T);
  switch (word) {
    case 16: return run_grad<T, 16 / S>(g, gy, out, st);
    case 8: return run_grad<T, 8 / S>(g, gy, out, st);
    case 4: return run_grad<T, 4 / S>(g, gy, out, st);
    default: return run_grad<T, 1>(g, gy, out, st);
  }
}

}  // namespace
}  // namespace kfac

using namespace kfac;

extern "C" int kfac_embedding(int dtype, const void* weight, int64_t vocab,
                              int width, const void* ids, int id_bytes, int64_t n,
                              int has_ignore, int64_t ignore, float scale,
                              void* out, void* stream) {
  int rc = check_ids("embedding", ids, id_bytes, n, vocab);
  if (rc == KFAC_OK) rc = check_rows("embedding", dtype, width);
  if (rc != KFAC_OK || n == 0) return rc;
  KFAC_REQUIRE(weight != nullptr && out != nullptr, "embedding: null pointer");
  const Ids s = make_ids(ids, id_bytes, n, vocab, has_ignore, ignore);
  const int word = word_bytes(weight, out, width, dtype);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == KFAC_WIRE_F32)
    return look_up_by<float>(word, weight, s, width, scale, out, st);
  if (dtype == KFAC_WIRE_F16)
    return look_up_by<__half>(word, weight, s, width, scale, out, st);
  return look_up_by<__nv_bfloat16>(word, weight, s, width, scale, out, st);
}

extern "C" size_t kfac_token_order_workspace_bytes(int64_t n, int64_t vocab) {
  if (n < 0 || vocab < 1) return 0;
  const SortPlan p = plan_sort(n, vocab);
  return 2 * p.keys + p.counts;
}

extern "C" int kfac_token_order(const void* ids, int id_bytes, int64_t n,
                                int64_t vocab, int has_ignore, int64_t ignore,
                                int* keys, int* positions, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const int rc = check_ids("token_order", ids, id_bytes, n, vocab);
  if (rc != KFAC_OK || n == 0) return rc;
  KFAC_REQUIRE(keys != nullptr && positions != nullptr,
               "token_order: null pointer");
  const SortPlan p = plan_sort(n, vocab);
  const size_t need = 2 * p.keys + p.counts;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(KFAC_ERR_WORKSPACE, "token_order: %zu bytes of workspace, %zu needed",
                workspace == nullptr ? (size_t)0 : workspace_bytes, need);
  KFAC_REQUIRE(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
               "token_order: the workspace is not aligned to 4 bytes");
  const Ids s = make_ids(ids, id_bytes, n, vocab, has_ignore, ignore);
  cudaStream_t st = (cudaStream_t)stream;
  if (p.tiles == 1) {
    const int smem = (int)sizeof(SortCounts) + kSortTile * 6;
    KFAC_CUDA(cudaFuncSetAttribute(token_sort_tile_kernel,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   smem));
    token_sort_tile_kernel<<<1, kSortThreads, smem, st>>>(s, p.bits, p.passes, keys,
                                                          positions);
    KFAC_LAUNCH_CHECK("token_sort_tile_kernel");
    return KFAC_OK;
  }
  char* ws = static_cast<char*>(workspace);
  int* spare_keys = reinterpret_cast<int*>(ws);
  int* spare_perm = reinterpret_cast<int*>(ws + p.keys);
  int* counts = reinterpret_cast<int*>(ws + 2 * p.keys);
  const unsigned tiles = (unsigned)p.tiles;
  const int *from_keys = nullptr, *from_perm = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    const Digit d = {pass * p.bits, (1 << p.bits) - 1};
    // (the last pass writes the caller's arrays)
    const bool out = ((p.passes - 1 - pass) & 1) == 0;
    int* to_keys = out ? keys : spare_keys;
    int* to_perm = out ? positions : spare_perm;
    token_count_kernel<<<tiles, kSortThreads, 0, st>>>(s, from_keys, d, counts);
    KFAC_LAUNCH_CHECK("token_count_kernel");
    if (p.tiles > kOwnBases) {
      token_bases_kernel<<<1, kSortThreads, 0, st>>>(counts, (int)tiles);
      KFAC_LAUNCH_CHECK("token_bases_kernel");
    }
    token_scatter_kernel<<<tiles, kSortThreads, 0, st>>>(
        s, from_keys, from_perm, d, counts, (int)tiles, to_keys, to_perm);
    KFAC_LAUNCH_CHECK("token_scatter_kernel");
    from_keys = to_keys;
    from_perm = to_perm;
  }
  return KFAC_OK;
}

extern "C" size_t kfac_embedding_grad_workspace_bytes(int64_t n, int width) {
  if (n < 0 || width < 1) return 0;
  // (the word's width changes how many chunks there are; the most)
  long long most = 0;
  for (int v = 1; v <= 8; v *= 2) {
    const GradPlan p = plan_grad(n, width, v);
    most = std::max(most, p.chunks * p.pitch);
  }
  return (size_t)most * 2 * sizeof(float);
}

extern "C" int kfac_embedding_grad(int dtype, const void* gy, int width,
                                   const int* keys, const int* positions,
                                   int64_t n, int64_t vocab, float scale,
                                   int accumulate, void* out, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  int rc = check_ids("embedding_grad", keys, 4, n, vocab);
  if (rc == KFAC_OK) rc = check_rows("embedding_grad", dtype, width);
  if (rc != KFAC_OK) return rc;
  KFAC_REQUIRE(out != nullptr && (n == 0 || (gy != nullptr && positions != nullptr)),
               "embedding_grad: null pointer");
  const size_t need = kfac_embedding_grad_workspace_bytes(n, width);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(KFAC_ERR_WORKSPACE,
                "embedding_grad: %zu bytes of workspace, %zu needed",
                workspace == nullptr ? (size_t)0 : workspace_bytes, need);
  KFAC_REQUIRE(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
               "embedding_grad: the workspace is not aligned to 16 bytes");
  Grad g = {};
  g.keys = keys;
  g.perm = positions;
  g.n = n;
  g.vocab = (int)vocab;
  g.width = width;
  g.part = static_cast<float*>(workspace);
  g.scale = scale;
  g.add = accumulate != 0;
  const int word = word_bytes(n == 0 ? out : gy, out, width, dtype);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == KFAC_WIRE_F32) return run_grad_by<float>(word, g, gy, out, st);
  if (dtype == KFAC_WIRE_F16) return run_grad_by<__half>(word, g, gy, out, st);
  return run_grad_by<__nv_bfloat16>(word, g, gy, out, st);
}

extern "C" size_t kfac_token_counts_workspace_bytes(int64_t vocab) {
  return vocab < 1 ? 0 : (size_t)vocab * sizeof(int);
}

extern "C" int kfac_token_counts(const void* ids, int id_bytes, int64_t n,
                                 int64_t vocab, int has_ignore, int64_t ignore,
                                 float alpha, float beta, float* out, float* mean,
                                 void* workspace, size_t workspace_bytes,
                                 void* stream) {
  const int rc = check_ids("token_counts", ids, id_bytes, n, vocab);
  if (rc != KFAC_OK) return rc;
  KFAC_REQUIRE(out != nullptr, "token_counts: null pointer");
  const size_t need = kfac_token_counts_workspace_bytes(vocab);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(KFAC_ERR_WORKSPACE, "token_counts: %zu bytes of workspace, %zu needed",
                workspace == nullptr ? (size_t)0 : workspace_bytes, need);
  KFAC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
               "token_counts: the workspace is not aligned to 4 bytes");
  int* counts = static_cast<int*>(workspace);
  cudaStream_t st = (cudaStream_t)stream;
  KFAC_CUDA(cudaMemsetAsync(counts, 0, need, st));
  if (n > 0) {
    const Ids s = make_ids(ids, id_bytes, n, vocab, has_ignore, ignore);
    token_histogram_kernel<<<(unsigned)std::min<long long>(ceil_div(n, 256), 8 * 148),
                             256, 0, st>>>(s, counts);
    KFAC_LAUNCH_CHECK("token_histogram_kernel");
  }
  token_counts_kernel<<<(unsigned)ceil_div(vocab, 256) + 1, 256, 0, st>>>(
      counts, (int)vocab, alpha, beta, out, mean);
  KFAC_LAUNCH_CHECK("token_counts_kernel");
  return KFAC_OK;
}
