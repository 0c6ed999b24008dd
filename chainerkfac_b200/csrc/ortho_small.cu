// Orthogonalised updates of small matrices: all steps of a matrix in one launch, with
// X, A and B in shared memory as planes of fp16 terms.  The same arithmetic as ortho.cu,
// which has the formulas; a launch of its own for each of its 15 products takes 9 us
// and more whatever the size.
//
// One block holds a matrix of sides up to 128 and 256.  A longer one is shared by the
// blocks of a cluster, 192 columns of the long side each: they add up A from their parts
// through distributed shared memory (every block sums some squares of 32 x 32, in the
// order of the blocks, and hands them to all), and compute B, each for itself.
//
// X lies in tiles of 128 rows x 64 columns, 128 bytes a row: the layout that the MMAs
// read as rows of k (A = X X^T) and as columns of k (B X) alike, so a step never moves
// X.  A matrix that is taller than wide is turned when it is read.  A sum is at most 256
// k long, with the cross terms of all of them first.
//
// Bound: latency.  Five steps: 64 x 147 32 us (15 launches 150), 128 x 256 57, 64 x 576
// 48, 128 x 1152 81 us.  (With an accumulator for every product of terms, which the MMAs
// do not need to stay apart, 36, 62, 50 and 86.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "ortho.cuh"
#include "planes.cuh"

namespace kfac {
namespace {

constexpr int OS_THREADS = 512;
constexpr int OS_WARPS = OS_THREADS / 32;
constexpr int OS_PLANE = 128 * 128;          // bytes: 128 rows of 64 fp16
constexpr int OS_TILE = 2 * OS_PLANE;        // hi, lo
constexpr int OS_UNIT = 32 * 32 * 4;         // bytes of a square of sums
// Tiles of X in a block; a cluster's blocks have 64 KB for the parts of A beside them.
__host__ __device__ constexpr int os_tiles(bool split) { return (split ? kSmallShare : kSmallLong) / 64; }
__host__ __device__ constexpr int os_smem(bool split) {
  return (os_tiles(split) + 2) * OS_TILE + (split ? 16 * OS_UNIT : 0) + 1024 + 1024;
}
static_assert(os_smem(false) <= 227 * 1024 && os_smem(true) <= 227 * 1024,
              "shared memory");
constexpr int kBlocksMax = kSmallClusterLong / kSmallShare;   // of a cluster
static_assert(kBlocksMax <= 16, "cluster size");

struct SmallControl {
  unsigned long long done;
  unsigned tmem_base;
  volatile int abort_flag;
};

// 16-byte word `word` of a row of 128 bytes.
__device__ __forceinline__ unsigned os_at(unsigned plane, int row, int word) {
  return plane + row * 128 + ((word ^ (row & 7)) << 4);
}

__device__ __forceinline__ void os_store16(unsigned addr, uint4 x) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x.x),
               "r"(x.y), "r"(x.z), "r"(x.w)
               : "memory");
}

// 32 x 32 values (in a PlaneTile's order) as terms: rows r0.., columns c0.. of planes
// in tiles of 64 columns.
__device__ __forceinline__ void os_put(unsigned planes, int r0, int c0, int lane,
                                       const float (&v)[32]) {
  unsigned hi[16], lo[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) pl_split2(v[2 * i], v[2 * i + 1], hi[i], lo[i]);
  const unsigned tile = planes + (c0 >> 6) * OS_TILE;
  const int row = r0 + lane, word = (c0 & 63) >> 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned at = os_at(tile, row, word + j);
    st_matrix(at, hi[2 * j], hi[2 * j + 1], hi[8 + 2 * j], hi[8 + 2 * j + 1]);
    st_matrix(at + OS_PLANE, lo[2 * j], lo[2 * j + 1], lo[8 + 2 * j],
              lo[8 + 2 * j + 1]);
  }
}

// v += beta * what is there.
__device__ __forceinline__ void os_add(unsigned planes, int r0, int c0, int lane,
                                       float beta, float (&v)[32]) {
  const unsigned tile = planes + (c0 >> 6) * OS_TILE;
  for (int term = 0; term < 2; ++term) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned x[4];
      ld_matrix(os_at(tile + term * OS_PLANE, r0 + lane, ((c0 & 63) >> 3) + j), x[0],
                x[1], x[2], x[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x[e]));
        const int at = 16 * (e >> 1) + 4 * j + 2 * (e & 1);
        v[at] = fmaf(beta, y.x, v[at]);
        v[at + 1] = fmaf(beta, y.y, v[at + 1]);
      }
    }
  }
}

// v = 32 x 32 of an accumulator.
__device__ __forceinline__ void os_sums(unsigned at, float (&v)[32]) {
  float x[16], y[16];
  tc_ld_16x32(at, x);
  tc_ld_16x32(at + (16u << 16), y);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    v[i] = x[i];
    v[16 + i] = y[i];
  }
}

__device__ __forceinline__ int parts_of(int a, int b) { return (a + b - 1) / b; }

template <typename T> __device__ __forceinline__ float value(T x);
template <> __device__ __forceinline__ float value(float x) { return x; }
template <> __device__ __forceinline__ float value(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float value(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded(float x) { return x; }
template <> __device__ __forceinline__ __half rounded(float x) {
  return __float2half_rn(x);
}
template <> __device__ __forceinline__ __nv_bfloat16 rounded(float x) {
  return __float2bfloat16_rn(x);
}

// SPLIT: a matrix by a cluster of l.blocks blocks.  A wait that runs out raises the
// status word and lets the others return at once; the block goes on to the end, so
// that the cluster's barriers have all their threads.
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(OS_THREADS, 1)
ortho_small_kernel(const __grid_constant__ SmallLaunch l) {
  int* const status = &g_plane_status;
  __shared__ double part[OS_WARPS];
  __shared__ double parts[16];               // of the cluster's blocks
  extern __shared__ unsigned char os_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(os_smem_raw) + 1023) & ~(uintptr_t)1023);
  SmallControl* ctl =
      reinterpret_cast<SmallControl*>(smem + os_smem(SPLIT) - 2048);
  const unsigned X = smem_u32(smem), A = X + os_tiles(SPLIT) * OS_TILE;
  const unsigned sums = A + 2 * OS_TILE;     // (SPLIT) parts of A: [slot][block]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int blocks = SPLIT ? l.blocks : 1;
  const int me = SPLIT ? (int)cluster_rank() : 0;
  const SmallJob job = l.j[blockIdx.x / blocks];
  const bool tall = job.rows > job.cols;
  const int r = tall ? job.cols : job.rows, length = tall ? job.rows : job.cols;
  // this block's columns of the long side (of a short matrix some have none)
  const int share = SPLIT ? (parts_of(length, blocks) + 63) & ~63 : length;
  const int first = min(me * share, length), c = min(share, length - first);
  const int xtiles = (c + 63) >> 6;

  if (warp == 0) {
    asm volatile(
        "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
        ::"r"(smem_u32(&ctl->tmem_base)), "r"(256)
        : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;"
                 ::: "memory");
    if (lane == 0) {
      mbar_init(&ctl->done, 1);
      ctl->abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  }

  if (SPLIT) cluster_sync();                 // all blocks are there to be written to

  // X = G / (|G| + eps), 2^13 times; zeros around it
  const T* const x = static_cast<const T*>(job.x);
  double sum = 0;
  // (a turned matrix's columns are whole rows in memory)
  const int count = r * c, width = SPLIT && !tall ? c : max(count, 1);
  const T* const from = x + (tall ? (long long)first * r : first);
  const int pitch = SPLIT && !tall ? length : width;
#pragma unroll 4
  for (int i = tid; i < count; i += OS_THREADS) {
    const double v = (double)value(from[(long long)(i / width) * pitch + i % width]);
    sum = fma(v, v, sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < OS_WARPS; ++w) sum += part[w];
  if constexpr (SPLIT) {
    if (tid < blocks)
      asm volatile("st.shared::cluster.f64 [%0], %1;"
                   ::"r"(cluster_addr(smem_u32(&parts[me]), tid)), "d"(sum)
                   : "memory");
    cluster_sync();
    sum = 0;
    for (int p = 0; p < blocks; ++p) sum += parts[p];
  }
  const double scale = (double)(1 << kXExp) / (sqrt(sum) + l.eps);
  const int words = 8 * xtiles;                 // of eight columns
#pragma unroll 1
  for (int i = tid; i < 128 * words; i += OS_THREADS) {
    // (neighbours read next to each other: along a row, or down the turned one's)
    const int row = tall ? i & 127 : i / words, word = tall ? i >> 7 : i % words;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = 8 * word + e;
      const long long at = tall ? (long long)(first + col) * r + row
                                : (long long)row * length + first + col;
      v[e] = row < r && col < c ? (float)((double)value(x[at]) * scale) : 0.f;
    }
    uint4 hi, lo;
    pl_split2(v[0], v[1], hi.x, lo.x);
    pl_split2(v[2], v[3], hi.y, lo.y);
    pl_split2(v[4], v[5], hi.z, lo.z);
    pl_split2(v[6], v[7], hi.w, lo.w);
    const unsigned to = os_at(X + (word >> 3) * OS_TILE, row, word & 7);
    os_store16(to, hi);
    os_store16(to + OS_PLANE, lo);
  }

  const int nk = (r + 15) >> 4, ck = (c + 15) >> 4;
  const int q = warp & 3, h = warp >> 2, r0 = 32 * q;
  unsigned phase = 0;
  unsigned tmem = 0, quarter = 0;
  // What every thread has written to shared memory is there for the MMAs; `issue` by
  // one of them; the accumulators are final.
  auto product = [&](auto issue) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem = ctl->tmem_base;
    quarter = tmem + ((unsigned)r0 << 16);
    if (warp == 0 && elect_one()) {
      issue();
      tc_commit(&ctl->done);
    }
    __syncwarp();
    mbar_wait_status(&ctl->done, phase, &ctl->abort_flag, status);
    __syncwarp();
    phase ^= 1;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  // planes times themselves over n times 16 k, cross terms first, while the sum is small
  auto square = [](unsigned tmem, unsigned planes, int n, unsigned idesc) {
    const unsigned long long lo = OS_PLANE >> 4;
    for (int k = 0; k < n; ++k) {
      const unsigned long long a =
          tc_smem_desc(planes + (k >> 2) * OS_TILE) + (k & 3) * 2;
      tc_mma_half(tmem, a, a + lo, idesc, k != 0);
      tc_mma_half(tmem, a + lo, a, idesc, 1);
    }
    for (int k = 0; k < n; ++k) {
      const unsigned long long a =
          tc_smem_desc(planes + (k >> 2) * OS_TILE) + (k & 3) * 2;
      tc_mma_half(tmem, a, a, idesc, 1);
    }
  };
  // of a sum of n additions that truncate, on average (see plane_gain)
  auto gain = [](int n) { return 1.f + 0.36f * (n + 1) * exp2f(-24); };

#pragma unroll 1
  for (int step = 0; step < l.steps; ++step) {
    const float* k3 = l.coefficients + 3 * step;
    // A = X X^T
    product([&]() {
      const unsigned idesc = tc_half_desc(16 * nk, false, false);
      square(tmem, X, ck, idesc);
    });
    const float make_a = exp2f(kAExp - 2 * kXExp) * gain(ck);
    const int squares = (r + 31) >> 5;       // a side of A, in units
    if (r0 < r) {
#pragma unroll 1
      for (int c0 = 32 * h; c0 < r; c0 += 32 * OS_WARPS / 4) {
        float v[32];
        os_sums(quarter + c0, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = ck > 0 ? v[i] * make_a : 0.f;
        if constexpr (!SPLIT) {
          os_put(A, r0, c0, lane, v);
        } else {
          const int unit = q * squares + (c0 >> 5);
          const unsigned to =
              cluster_addr(sums + (unit / blocks * blocks + me) * OS_UNIT + lane * 16,
                           unit % blocks);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            cluster_store(to + 512 * i, v[4 * i], v[4 * i + 1], v[4 * i + 2],
                          v[4 * i + 3]);
        }
      }
    }
    if constexpr (SPLIT) {
      cluster_sync();           // the parts are there, and no block needs its B
#pragma unroll 1
      for (int slot = warp; slot * blocks + me < squares * squares; slot += OS_WARPS) {
        const int unit = slot * blocks + me, u0 = unit / squares * 32;
        const int c0 = unit % squares * 32;
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
#pragma unroll 1
        for (int p = 0; p < blocks; ++p) {
          const unsigned at = sums + (slot * blocks + p) * OS_UNIT + lane * 16;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float4 y;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w)
                         : "r"(at + 512 * i)
                         : "memory");
            v[4 * i] += y.x;
            v[4 * i + 1] += y.y;
            v[4 * i + 2] += y.z;
            v[4 * i + 3] += y.w;
          }
        }
        os_put(A, u0, c0, lane, v);
        __syncwarp();
        const unsigned tile = A + (c0 >> 6) * OS_TILE;
        for (int term = 0; term < 2; ++term) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned at =
                os_at(tile + term * OS_PLANE, u0 + lane, ((c0 & 63) >> 3) + j);
            float4 y;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w)
                         : "r"(at)
                         : "memory");
            for (int p = 0; p < blocks; ++p)
              if (p != me) cluster_store(cluster_addr(at, p), y.x, y.y, y.z, y.w);
          }
        }
      }
      cluster_sync();                        // every block has all of A
    }
    // B = a I + b A + c A A, in A's place
    product([&]() {
      const unsigned idesc = tc_half_desc(16 * nk, false, false);
      square(tmem, A, nk, idesc);
    });
    const float cube = k3[2] * exp2f(-kAExp) * gain(nk), diag = k3[0] * exp2f(kAExp);
    if (r0 < r) {
#pragma unroll 1
      for (int c0 = 32 * h; c0 < r; c0 += 32 * OS_WARPS / 4) {
        float v[32];
        os_sums(quarter + c0, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= cube;
        os_add(A, r0, c0, lane, k3[1], v);
        if (c0 == r0) {
          const int d = 2 * (lane & 3) - (lane >> 2);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int row = 16 * (i >> 4) + 8 * ((i >> 1) & 1);
            if (row - 8 * ((i >> 2) & 3) - (i & 1) == d &&
                r0 + row + (lane >> 2) < r)
              v[i] += diag;
          }
        }
        os_put(A, r0, c0, lane, v);
      }
    }
    // X = B X
    product([&]() {
      if (SPLIT && ck == 0) return;
      const unsigned idesc = tc_half_desc(16 * ck, false, true);
      for (int k = 0; k < nk; ++k) {
        const unsigned long long a =
            tc_smem_desc(A + (k >> 2) * OS_TILE) + (k & 3) * 2;
        const unsigned long long b = tc_smem_desc_mn(X + k * 2048, OS_TILE);
        const unsigned long long lo = OS_PLANE >> 4;
        tc_mma_half(tmem, a, b + lo, idesc, k != 0);
        tc_mma_half(tmem, a + lo, b, idesc, 1);
      }
      for (int k = 0; k < nk; ++k)
        tc_mma_half(tmem, tc_smem_desc(A + (k >> 2) * OS_TILE) + (k & 3) * 2,
                    tc_smem_desc_mn(X + k * 2048, OS_TILE), idesc, 1);
    });
    const bool last = step + 1 == l.steps;
    const float make_x =
        exp2f(last ? -(kXExp + kAExp) : -kAExp) * gain(nk) * (last ? job.scale : 1.f);
    if (r0 >= r) continue;
#pragma unroll 1
    for (int c0 = 32 * h; c0 < c; c0 += 32 * OS_WARPS / 4) {
      float v[32];
      os_sums(quarter + c0, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= make_x;
      if (!last) {
        os_put(X, r0, c0, lane, v);
        continue;
      }
      // out through this warp's 4 KB of what was A
      const unsigned piece = A + warp * 4096;
      T* const dst = static_cast<T*>(job.dst);
      T* const param = static_cast<T*>(job.param);
      __syncwarp();
      pl_put_floats(piece, v, lane);
      __syncwarp();
      const int rows = min(32, r - r0), cols = min(32, c - c0);
      // along a row of the result: columns, or the turned matrix's rows
      const int lines = tall ? cols : rows, in = tall ? rows : cols;
      const long long at0 = tall ? (long long)(first + c0) * r + r0
                                 : (long long)r0 * length + first + c0;
      const int pitch = tall ? r : length;
#pragma unroll 4
      for (int i = 0; i < lines; ++i) {
        const float y = tall ? pl_float(piece, lane, i) : pl_float(piece, i, lane);
        const long long at = at0 + (long long)i * pitch + lane;
        if (lane < in && dst != nullptr) dst[at] = rounded<T>(y);
        if (lane < in && param != nullptr)
          param[at] = rounded<T>(fmaf(l.keep, value(param[at]), -l.lr * y));
      }
      __syncwarp();
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) tc_release(ctl->tmem_base, 256u, ctl->abort_flag != 0);
}

template <typename T, bool SPLIT>
int launch_as(const SmallLaunch& l, cudaStream_t st) {
  auto* kernel = ortho_small_kernel<T, SPLIT>;
  static std::mutex mu;
  static bool done[64] = {false};
  int dev = 0;
  KFAC_CUDA(cudaGetDevice(&dev));
  KFAC_REQUIRE(dev >= 0 && dev < 64, "device index %d unsupported", dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      KFAC_CUDA(cudaFuncSetAttribute(
          kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, os_smem(SPLIT)));
      if (SPLIT)
        KFAC_CUDA(cudaFuncSetAttribute(
            kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      done[dev] = true;
    }
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = l.blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(l.n * l.blocks);
  cfg.blockDim = dim3(OS_THREADS);
  cfg.dynamicSmemBytes = os_smem(SPLIT);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 1 : 0;
  KFAC_CUDA(cudaLaunchKernelEx(&cfg, kernel, l));
  KFAC_LAUNCH_CHECK("ortho_small_kernel");
  return KFAC_OK;
}

template <typename T>
int launch_of(const SmallLaunch& l, cudaStream_t st) {
  return l.blocks > 1 ? launch_as<T, true>(l, st) : launch_as<T, false>(l, st);
}

}  // namespace

int launch_ortho_small(SmallLaunch& l, int dtype, cudaStream_t st) {
  if (l.n == 0) return KFAC_OK;
  // one block for each matrix if all are that short, else as many as the longest one
  // takes; powers of two, which fill the clusters that the GPU has room for
  int longest = 0;
  for (int i = 0; i < l.n; ++i)
    longest = std::max(longest, std::max(l.j[i].rows, l.j[i].cols));
  l.blocks = 1;
  if (longest > kSmallLong)
    while (l.blocks < kBlocksMax && l.blocks * kSmallShare < longest) l.blocks *= 2;
  if (dtype == KFAC_WIRE_F32) return launch_of<float>(l, st);
  if (dtype == KFAC_WIRE_F16) return launch_of<__half>(l, st);
  return launch_of<__nv_bfloat16>(l, st);
}

int ortho_small_status_read(int* out) {
  KFAC_CUDA(cudaMemcpyFromSymbol(out, g_plane_status, sizeof(int)));
  return KFAC_OK;
}

}  // namespace kfac
