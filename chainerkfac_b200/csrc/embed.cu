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
#include <initializer_list>

#include "common.cuh"
#include "tc_common.cuh"

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

// A word to memory, past the caches' other contents where what is written is more
// than they hold anyway (STREAM).
template <bool STREAM, typename P>
__device__ __forceinline__ void put_word(P* to, const P& x) {
  if constexpr (STREAM && sizeof(P) == 16) {
    __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&x));
  } else {
    *to = x;
  }
}
constexpr long long kStreamBytes = 64LL << 20;      // half of the L2 cache

// ------------------------------------------------------------------ lookup

// 65536 tokens x 2048 bf16 over 128000: 66 us (a copy of as much takes 88), 70 with four
// rows in flight; 72 with 128 threads, 88 with 256, 119 with 256, four rows and stores
// that stay in the caches.
constexpr int kLookThreads = 64;
constexpr int kLookRows = 2;      // rows a thread has in flight
// And words of each, more of narrow ones: 32768 x 1023 fp32 41 us, with one 57.
__host__ __device__ constexpr int look_words(int bytes) {
  return bytes == 16 ? 1 : bytes == 8 ? 2 : 4;
}

// `lanes` threads (a power of two) share a row; a block has kLookThreads / lanes
// rows at a time, kLookRows times.
template <typename T, int V, bool STREAM>
__global__ void __launch_bounds__(kLookThreads)
embed_lookup_kernel(const T* __restrict__ weight, const Ids ids, int width,
                    float scale, T* __restrict__ out, int lanes) {
  using P = Pack<T, V>;
  constexpr int kWords = look_words(V * (int)sizeof(T));
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
    for (int w0 = at; w0 < words; w0 += kWords * lanes) {
      P x[kLookRows][kWords];
#pragma unroll
      for (int u = 0; u < kLookRows; ++u)
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          const int w = w0 + k * lanes;
          if (row[u] >= 0 && (kWords == 1 || w < words))
            x[u][k] = *reinterpret_cast<const P*>(
                weight + (long long)row[u] * width + (long long)w * V);
        }
#pragma unroll
      for (int u = 0; u < kLookRows; ++u) {
        const long long i = i0 + (long long)u * per + sub;
        if (i >= ids.n) continue;
        const float none = row[u] == kIgnored ? 0.f : __int_as_float(0x7fc00000);
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          const int w = w0 + k * lanes;
          if (kWords > 1 && w >= words) break;
#pragma unroll
          for (int e = 0; e < V; ++e)
            x[u][k].x[e] = Num<T>::put(
                row[u] >= 0 ? scale * Num<T>::get(x[u][k].x[e]) : none);
          put_word<STREAM>(
              reinterpret_cast<P*>(out + i * width + (long long)w * V), x[u][k]);
        }
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
// warp's counts.  (Keys behind the end have all bits set and come last.)
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

// All passes of up to 131072 tokens in one launch, by a cluster of up to sixteen blocks:
// a block holds 1024 ITEMS keys, hands its counts to the others and puts every key
// where it belongs in any block's shared memory.  65536 tokens of 128000: 26 us (with
// two launches a pass 42), 12345 of 32003 14 us (37).
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int kClusterItems = 8;
constexpr int kClusterMax = 16;
constexpr int kClusterTokens = kClusterMax * kClusterThreads * kClusterItems;

struct ClusterCounts {
  unsigned short warp[kClusterWarps][kBins];
  int total[kBins];
  int base[kBins];
  int part[kClusterWarps];
};

__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned in_block(const void* p, int block) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(r)
      : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(block));
  return r;
}

template <int ITEMS>
__global__ void __launch_bounds__(kClusterThreads)
token_sort_cluster_kernel(const Ids ids, int bits, int passes, int* keys_out,
                          int* perm_out) {
  extern __shared__ __align__(16) unsigned char sort_smem[];
  ClusterCounts& s = *reinterpret_cast<ClusterCounts*>(sort_smem);
  int2* const data = reinterpret_cast<int2*>(sort_smem + sizeof(ClusterCounts));
  constexpr int kTile = kClusterThreads * ITEMS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = gridDim.x, me = blockIdx.x;      // (the launch is one cluster)
  const int first = warp * 32 * ITEMS + lane, n = (int)ids.n;
  int key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    pos[j] = me * kTile + first + 32 * j;
    // (a key behind the end has all bits set: it stays behind all others)
    key[j] = pos[j] < n ? key_of(ids, pos[j]) : 0x7fffffff;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const Digit d = {pass * bits, (1 << bits) - 1};
    unsigned short* const mine = s.warp[warp];
    for (int b = lane; b < kBins / 2; b += 32)
      reinterpret_cast<unsigned*>(mine)[b] = 0;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int digit = (key[j] >> d.shift) & d.mask;
      const unsigned peers = __match_any_sync(0xffffffffu, digit);
      const int before = mine[digit];
      __syncwarp();
      rank[j] = before + __popc(peers & ((1u << lane) - 1));
      if (lane == 31 - __clz(peers))
        mine[digit] = (unsigned short)(before + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
      int run = 0;
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) {
        const int c = s.warp[w][threadIdx.x];
        s.warp[w][threadIdx.x] = (unsigned short)run;
        run += c;
      }
      s.total[threadIdx.x] = run;
    }
    cluster_barrier();
    int all = 0, before = 0;
    if (threadIdx.x < kBins) {
      int x[kClusterMax];                    // (all on their way at once)
#pragma unroll
      for (int c = 0; c < kClusterMax; ++c) {
        x[c] = 0;
        if (c < blocks)
          asm volatile("ld.shared::cluster.s32 %0, [%1];"
                       : "=r"(x[c])
                       : "r"(in_block(&s.total[threadIdx.x], c)));
      }
#pragma unroll
      for (int c = 0; c < kClusterMax; ++c) {
        all += x[c];
        before += c < me ? x[c] : 0;
      }
    }
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s.part[warp] = inc;
    __syncthreads();
    if (threadIdx.x < kBins) {
      int front = 0;
#pragma unroll
      for (int w = 0; w < kBins / 32; ++w) front += w < warp ? s.part[w] : 0;
      s.base[threadIdx.x] = front + inc - all + before;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int digit = (key[j] >> d.shift) & d.mask;
      const int to = s.base[digit] + s.warp[warp][digit] + rank[j];
      asm volatile("st.shared::cluster.v2.s32 [%0], {%1, %2};"
                   ::"r"(in_block(&data[to % kTile], to / kTile)), "r"(key[j]),
                     "r"(pos[j])
                   : "memory");
    }
    cluster_barrier();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int2 x = data[first + 32 * j];
      key[j] = x.x;
      pos[j] = x.y;
    }
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int i = me * kTile + first + 32 * j;
    if (i < n) {
      keys_out[i] = key[j];
      perm_out[i] = pos[j];
    }
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

template <typename T, int V, bool STREAM = false>
__device__ __forceinline__ void put_row(T* out, const float (&acc)[V], float scale,
                                        bool add) {
  using P = Pack<T, V>;
  P x;
  if (add) x = *reinterpret_cast<const P*>(out);
#pragma unroll
  for (int e = 0; e < V; ++e)
    x.x[e] = Num<T>::put(add ? fmaf(scale, acc[e], Num<T>::get(x.x[e]))
                             : scale * acc[e]);
  put_word<STREAM>(reinterpret_cast<P*>(out), x);
}

template <typename T, int V, bool STREAM>
__global__ void __launch_bounds__(kGradThreads)
embed_grad_kernel(const Grad g, const T* gy, T* out) {
  using P = Pack<T, V>;
  constexpr int kGradAhead = 8;      // rows in flight
  let_next_launch_begin();
  wait_for_launch_before();
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
    // (rows next to each other as one piece of memory, whatever their width: 32003
    // rows of 771 floats 33 us, row by row in words of four bytes 36)
    unsigned rows = clear;
    while (rows != 0) {
      const int r = __ffs(rows) - 1;
      const unsigned run = ~(rows >> r);
      const int many = run == 0 ? 32 - r : min(__ffs(run) - 1, 32 - r);
      rows = r + many >= 32 ? 0 : rows & (~0u << (r + many));
      char* to = reinterpret_cast<char*>(out + (long long)(r0 + r) * g.width);
      const long long bytes = (long long)many * g.width * sizeof(T);
      const int front = (int)min(bytes, (long long)(-reinterpret_cast<uintptr_t>(to) & 15));
      const long long words = (bytes - front) >> 4;
      uint4* const body = reinterpret_cast<uint4*>(to + front);
      const int back = (int)(bytes - front - (words << 4));
      const T none = Num<T>::put(0.f);
      constexpr int S = sizeof(T);
      if (S * (int)threadIdx.x < front) reinterpret_cast<T*>(to)[threadIdx.x] = none;
      if (S * (int)threadIdx.x < back)
        reinterpret_cast<T*>(body + words)[threadIdx.x] = none;
      for (long long w = threadIdx.x; w < words; w += kGradThreads)
        put_word<STREAM>(body + w, make_uint4(0, 0, 0, 0));
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
      put_row<T, V, STREAM>(out + (long long)cur * g.width + col, acc, g.scale, g.add);
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

// Tokens whose positions lie in several chunks: the sum of their parts, in order, by
// the block of the chunk where the token begins; four columns a thread.  (A block for
// every 128 columns of a chunk, most of them with nothing to do, took 75 us for 65536
// tokens x 2048, so 14.)
constexpr int kJoinThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
embed_join_kernel(const Grad g, T* out) {
  __shared__ long long s_end;
  const long long chunk = blockIdx.x;
  const long long p0 = chunk * g.chunk, p1 = p0 + g.chunk;
  if (p1 >= g.n) return;
  wait_for_launch_before();
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
    s_end = (lo - 1) / g.chunk + 1;      // first chunk without it
  }
  __syncthreads();
  const long long end = s_end;
  const float4* const part = reinterpret_cast<const float4*>(g.part);
  const long long pitch = g.pitch >> 2;
  for (int c = threadIdx.x; 4 * c < g.width; c += kJoinThreads) {
    float4 sum = part[(2 * chunk + 1) * pitch + c];
#pragma unroll 8
    for (long long k = chunk + 1; k < end; ++k) {
      const float4 x = part[2 * k * pitch + c];
      sum.x += x.x;
      sum.y += x.y;
      sum.z += x.z;
      sum.w += x.w;
    }
    const float all[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float acc[1] = {all[e]};
      if (4 * c + e < g.width)
        put_row<T, 1>(out + (long long)key * g.width + 4 * c + e, acc, g.scale, g.add);
    }
  }
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
  KFAC_REQUIRE(aligned_to(ids, id_bytes), "%s: tokens not aligned to %d bytes", what,
               id_bytes);
  return KFAC_OK;
}

int check_rows(const char* what, int dtype, int width) {
  KFAC_REQUIRE(dtype == KFAC_WIRE_F32 || dtype == KFAC_WIRE_F16 ||
                   dtype == KFAC_WIRE_BF16,
               "%s: unknown element type %d", what, dtype);
  KFAC_REQUIRE(width >= 1 && width <= (1 << 28), "%s: rows of %d values (1 .. 2^28)",
               what, width);
  return KFAC_OK;
}

// Pieces of memory that a call reads, or writes besides.
struct Piece {
  const void* p;
  size_t bytes;
};
int check_apart(const char* what, Piece out, std::initializer_list<Piece> others) {
  for (const Piece& o : others)
    KFAC_REQUIRE(!overlap(out.p, out.bytes, o.p, o.bytes),
                 "%s: what is written overlaps another array", what);
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
  const bool stream = ids.n * width * (long long)sizeof(T) > kStreamBytes;
  auto* kernel = stream ? embed_lookup_kernel<T, V, true>
                        : embed_lookup_kernel<T, V, false>;
  kernel<<<(unsigned)std::min<long long>(blocks, 1 << 20), kLookThreads, 0, st>>>(
      static_cast<const T*>(weight), ids, width, scale, static_cast<T*>(out), lanes);
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

// (up to 2048 tokens by one block: a cluster's barriers take longer than its help)
template <int ITEMS>
int launch_sort(const Ids& s, const SortPlan& p, int blocks, int* keys, int* positions,
                cudaStream_t st) {
  const int smem = (int)sizeof(ClusterCounts) + kClusterThreads * ITEMS * 8;
  if (smem > 48 * 1024)
    KFAC_CUDA(cudaFuncSetAttribute(token_sort_cluster_kernel<ITEMS>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (blocks > 8)
    KFAC_CUDA(cudaFuncSetAttribute(token_sort_cluster_kernel<ITEMS>,
                                   cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KFAC_CUDA(cudaLaunchKernelEx(&cfg, token_sort_cluster_kernel<ITEMS>, s, p.bits,
                               p.passes, keys, positions));
  KFAC_LAUNCH_CHECK("token_sort_cluster_kernel");
  return KFAC_OK;
}

int sort_in_cluster(const Ids& s, const SortPlan& p, int* keys, int* positions,
                    cudaStream_t st) {
  constexpr int T = kClusterThreads;
  if (s.n <= T) return launch_sort<1>(s, p, 1, keys, positions, st);
  if (s.n <= 2 * T) return launch_sort<2>(s, p, 1, keys, positions, st);
  if (s.n <= 8 * T) return launch_sort<1>(s, p, 8, keys, positions, st);
  if (s.n <= 16 * T) return launch_sort<1>(s, p, 16, keys, positions, st);
  if (s.n <= 32 * T) return launch_sort<2>(s, p, 16, keys, positions, st);
  if (s.n <= 64 * T) return launch_sort<4>(s, p, 16, keys, positions, st);
  return launch_sort<8>(s, p, 16, keys, positions, st);
}

SortPlan plan_sort(int64_t n, int64_t vocab) {
  SortPlan p;
  int need = 1;
  while (need < 31 && (vocab >> need) != 0) ++need;      // keys 0 .. vocab
  p.passes = (need + kDigitBits - 1) / kDigitBits;
  p.bits = (need + p.passes - 1) / p.passes;
  p.tiles = (n + kSortTile - 1) / kSortTile;
  p.keys = n > kClusterTokens ? ((size_t)n * 4 + 255) & ~(size_t)255 : 0;
  p.counts = n > kClusterTokens ? (size_t)p.tiles * kBins * sizeof(int) : 0;
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
  while (p.chunk < 256 &&
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
  const bool stream =
      !g.add && (long long)g.vocab * g.width * (long long)sizeof(T) > kStreamBytes;
  auto* kernel = stream ? embed_grad_kernel<T, V, true> : embed_grad_kernel<T, V, false>;
  const int rc = launch_behind("embed_grad_kernel", true, kernel, (int)blocks,
                               kGradThreads, 0, st, g, static_cast<const T*>(gy),
                               static_cast<T*>(out));
  if (rc != KFAC_OK) return rc;
  if (p.chunks > 1) {
    KFAC_REQUIRE(p.chunks < (1LL << 31), "embedding_grad: too many blocks");
    return launch_behind("embed_join_kernel", true, embed_join_kernel<T>, (int)p.chunks,
                         kJoinThreads, 0, st, g, static_cast<T*>(out));
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
  const size_t size = type_size(dtype);
  KFAC_REQUIRE(aligned_to(weight, size) && aligned_to(out, size),
               "embedding: rows not aligned to their type");
  rc = check_apart("embedding", {out, (size_t)n * width * size},
                   {{weight, (size_t)vocab * width * size}, {ids, (size_t)n * id_bytes}});
  if (rc != KFAC_OK) return rc;
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
  int rc = check_ids("token_order", ids, id_bytes, n, vocab);
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
  KFAC_REQUIRE(aligned_to(keys, 4) && aligned_to(positions, 4),
               "token_order: keys or positions not aligned to 4 bytes");
  const size_t bytes = (size_t)n * 4;
  rc = check_apart("token_order", {keys, bytes},
                   {{positions, bytes}, {ids, (size_t)n * id_bytes}, {workspace, need}});
  if (rc == KFAC_OK)
    rc = check_apart("token_order", {positions, bytes},
                     {{ids, (size_t)n * id_bytes}, {workspace, need}});
  if (rc != KFAC_OK) return rc;
  const Ids s = make_ids(ids, id_bytes, n, vocab, has_ignore, ignore);
  cudaStream_t st = (cudaStream_t)stream;
  if (n <= kClusterTokens) return sort_in_cluster(s, p, keys, positions, st);
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
  const size_t size = type_size(dtype), tokens = (size_t)n * 4;
  KFAC_REQUIRE(aligned_to(gy, size) && aligned_to(out, size) && aligned_to(positions, 4),
               "embedding_grad: arrays not aligned to their types");
  rc = check_apart("embedding_grad", {out, (size_t)vocab * width * size},
                   {{gy, (size_t)n * width * size}, {keys, tokens}, {positions, tokens},
                    {workspace, need}});
  if (rc != KFAC_OK) return rc;
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
  int rc = check_ids("token_counts", ids, id_bytes, n, vocab);
  if (rc != KFAC_OK) return rc;
  KFAC_REQUIRE(out != nullptr, "token_counts: null pointer");
  const size_t need = kfac_token_counts_workspace_bytes(vocab);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(KFAC_ERR_WORKSPACE, "token_counts: %zu bytes of workspace, %zu needed",
                workspace == nullptr ? (size_t)0 : workspace_bytes, need);
  KFAC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
               "token_counts: the workspace is not aligned to 4 bytes");
  KFAC_REQUIRE(aligned_to(out, 4) && aligned_to(mean, 4),
               "token_counts: counts not aligned to 4 bytes");
  const Piece tokens = {ids, (size_t)n * id_bytes}, scratch = {workspace, need};
  rc = check_apart("token_counts", {out, (size_t)vocab * 4},
                   {tokens, scratch, {mean, sizeof(float)}});
  if (rc == KFAC_OK)
    rc = check_apart("token_counts", {mean, sizeof(float)}, {tokens, scratch});
  if (rc != KFAC_OK) return rc;
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
