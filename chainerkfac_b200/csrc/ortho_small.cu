// Orthogonalised updates of small matrices (sides of up to 128 and 256): all steps of a
// matrix by one block, with X, A and B in shared memory as planes of fp16 terms.  The
// same arithmetic as ortho.cu, which has the formulas; a launch of its own for each of
// its 15 products takes 9 us whatever the size.
//
// X lies in tiles of 128 rows x 64 columns, 128 bytes a row: the layout that the MMAs
// read as rows of k (A = X X^T) and as columns of k (B X) alike, so a step never moves
// X.  A matrix that is taller than wide is turned when it is read.  Every product of
// terms has an accumulator of its own (A's lo * hi and hi * lo as well), so that the MMAs
// do not wait for each other; a sum is at most 256 k long.
//
// Bound: latency.  SMALLTIMES
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
constexpr int OS_XTILES = kSmallLong / 64;
constexpr int OS_SMEM = OS_XTILES * OS_TILE + 2 * OS_TILE + 1024 + 1024;
static_assert(OS_SMEM <= 227 * 1024, "shared memory");

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
                                       const float (&v)[32], int terms) {
  unsigned hi[16], lo[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) pl_split2(v[2 * i], v[2 * i + 1], hi[i], lo[i]);
  const unsigned tile = planes + (c0 >> 6) * OS_TILE;
  const int row = r0 + lane, word = (c0 & 63) >> 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned at = os_at(tile, row, word + j);
    st_matrix(at, hi[2 * j], hi[2 * j + 1], hi[8 + 2 * j], hi[8 + 2 * j + 1]);
    if (terms == 2)
      st_matrix(at + OS_PLANE, lo[2 * j], lo[2 * j + 1], lo[8 + 2 * j],
                lo[8 + 2 * j + 1]);
  }
}

// v += beta * what is there.
__device__ __forceinline__ void os_add(unsigned planes, int r0, int c0, int lane,
                                       float beta, float (&v)[32], int terms) {
  const unsigned tile = planes + (c0 >> 6) * OS_TILE;
  for (int term = 0; term < terms; ++term) {
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

// v = the sum of `n` accumulators 32 x 32, `apart` columns from each other.
__device__ __forceinline__ void os_sums(unsigned at, int n, int apart, float (&v)[32]) {
  float x[16], y[16];
  tc_ld_16x32(at, x);
  tc_ld_16x32(at + (16u << 16), y);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    v[i] = x[i];
    v[16 + i] = y[i];
  }
#pragma unroll 1
  for (int k = 1; k < n; ++k) {
    tc_ld_16x32(at + k * apart, x);
    tc_ld_16x32(at + k * apart + (16u << 16), y);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] += x[i];
      v[16 + i] += y[i];
    }
  }
}

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

template <typename T>
__global__ void __launch_bounds__(OS_THREADS, 1)
ortho_small_kernel(const __grid_constant__ SmallLaunch l) {
  int* const status = &g_plane_status;
  __shared__ double part[OS_WARPS];
  extern __shared__ unsigned char os_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(os_smem_raw) + 1023) & ~(uintptr_t)1023);
  SmallControl* ctl =
      reinterpret_cast<SmallControl*>(smem + (OS_XTILES + 2) * OS_TILE);
  const unsigned X = smem_u32(smem), A = X + OS_XTILES * OS_TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const SmallJob job = l.j[blockIdx.x];
  const bool tall = job.rows > job.cols;
  const int r = tall ? job.cols : job.rows, c = tall ? job.rows : job.cols;
  const int xtiles = (c + 63) >> 6;

  if (warp == 0) {
    asm volatile(
        "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
        ::"r"(smem_u32(&ctl->tmem_base)), "r"(512)
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

  // X = G / (|G| + eps), 2^13 times; zeros around it
  const T* const x = static_cast<const T*>(job.x);
  double sum = 0;
  const int count = r * c;
#pragma unroll 4
  for (int i = tid; i < count; i += OS_THREADS) {
    const double v = (double)value(x[i]);
    sum = fma(v, v, sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < OS_WARPS; ++w) sum += part[w];
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
      const int at = tall ? col * r + row : row * c + col;
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

  const int terms = sizeof(T) == 4 ? 2 : 1;     // of A and B
  const int nk = (r + 15) >> 4, ck = (c + 15) >> 4;
  const int q = warp & 3, h = warp >> 2, r0 = 32 * q;
  unsigned phase = 0;
  bool ok = true;
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
    ok = mbar_wait_status(&ctl->done, phase, &ctl->abort_flag, status);
    ok = __syncthreads_and(ok);            // all of the block go on, or none
    phase ^= 1;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  // of a sum of n additions that truncate, on average (see plane_gain)
  auto gain = [](int n) { return 1.f + 0.36f * (n + 1) * exp2f(-24); };

#pragma unroll 1
  for (int step = 0; step < l.steps && ok; ++step) {
    const float* k3 = l.coefficients + 3 * step;
    // A = X X^T
    product([&]() {
      const unsigned idesc = tc_half_desc(16 * nk, false, false);
      for (int k = 0; k < ck; ++k) {
        const unsigned long long a =
            tc_smem_desc(X + (k >> 2) * OS_TILE) + (k & 3) * 2;
        const unsigned long long lo = OS_PLANE >> 4;
        tc_mma_half(tmem, a, a, idesc, k != 0);
        if (terms == 2) {
          tc_mma_half(tmem + 128, a, a + lo, idesc, k != 0);
          tc_mma_half(tmem + 256, a + lo, a, idesc, k != 0);
        }
      }
    });
    if (!ok) break;
    const float make_a = exp2f(kAExp - 2 * kXExp) * gain(ck);
    if (r0 < r) {
#pragma unroll 1
      for (int c0 = 32 * h; c0 < r; c0 += 32 * OS_WARPS / 4) {
        float v[32];
        os_sums(quarter + c0, 2 * terms - 1, 128, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= make_a;
        os_put(A, r0, c0, lane, v, terms);
      }
    }
    // B = a I + b A + c A A, in A's place
    product([&]() {
      const unsigned idesc = tc_half_desc(16 * nk, false, false);
      for (int k = 0; k < nk; ++k) {
        const unsigned long long a =
            tc_smem_desc(A + (k >> 2) * OS_TILE) + (k & 3) * 2;
        const unsigned long long lo = OS_PLANE >> 4;
        tc_mma_half(tmem, a, a, idesc, k != 0);
        if (terms == 2) {
          tc_mma_half(tmem + 128, a, a + lo, idesc, k != 0);
          tc_mma_half(tmem + 256, a + lo, a, idesc, k != 0);
        }
      }
    });
    if (!ok) break;
    const float square = k3[2] * exp2f(-kAExp) * gain(nk), diag = k3[0] * exp2f(kAExp);
    if (r0 < r) {
#pragma unroll 1
      for (int c0 = 32 * h; c0 < r; c0 += 32 * OS_WARPS / 4) {
        float v[32];
        os_sums(quarter + c0, 2 * terms - 1, 128, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= square;
        os_add(A, r0, c0, lane, k3[1], v, terms);
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
        os_put(A, r0, c0, lane, v, terms);
      }
    }
    // X = B X
    product([&]() {
      const unsigned idesc = tc_half_desc(16 * ck, false, true);
      for (int k = 0; k < nk; ++k) {
        const unsigned long long a =
            tc_smem_desc(A + (k >> 2) * OS_TILE) + (k & 3) * 2;
        const unsigned long long b = tc_smem_desc_mn(X + k * 2048, OS_TILE);
        const unsigned long long lo = OS_PLANE >> 4;
        tc_mma_half(tmem, a, b, idesc, k != 0);
        tc_mma_half(tmem + 256, a, b + lo, idesc, k != 0);
        if (terms == 2) tc_mma_half(tmem + 256, a + lo, b, idesc, 1);
      }
    });
    if (!ok) break;
    const bool last = step + 1 == l.steps;
    const float make_x =
        exp2f(last ? -(kXExp + kAExp) : -kAExp) * gain(nk) * (last ? job.scale : 1.f);
    if (r0 >= r) continue;
#pragma unroll 1
    for (int c0 = 32 * h; c0 < c; c0 += 32 * OS_WARPS / 4) {
      float v[32];
      os_sums(quarter + c0, 2, 256, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= make_x;
      if (!last) {
        os_put(X, r0, c0, lane, v, 2);
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
      const long long at0 = tall ? (long long)c0 * r + r0 : (long long)r0 * c + c0;
      const int pitch = tall ? r : c;
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
  if (warp == 0) tc_release(ctl->tmem_base, 512u, ctl->abort_flag != 0);
}

template <typename T>
int launch_as(const SmallLaunch& l, cudaStream_t st) {
  static std::mutex mu;
  static bool done[64] = {false};
  int dev = 0;
  KFAC_CUDA(cudaGetDevice(&dev));
  KFAC_REQUIRE(dev >= 0 && dev < 64, "device index %d unsupported", dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      KFAC_CUDA(cudaFuncSetAttribute(ortho_small_kernel<T>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     OS_SMEM));
      done[dev] = true;
    }
  }
  ortho_small_kernel<T><<<l.n, OS_THREADS, OS_SMEM, st>>>(l);
  KFAC_LAUNCH_CHECK("ortho_small_kernel");
  return KFAC_OK;
}

}  // namespace

int launch_ortho_small(const SmallLaunch& l, int dtype, cudaStream_t st) {
  if (l.n == 0) return KFAC_OK;
  if (dtype == KFAC_WIRE_F32) return launch_as<float>(l, st);
  if (dtype == KFAC_WIRE_F16) return launch_as<__half>(l, st);
  return launch_as<__nv_bfloat16>(l, st);
}

int ortho_small_status_read(int* out) {
  KFAC_CUDA(cudaMemcpyFromSymbol(out, g_plane_status, sizeof(int)));
  return KFAC_OK;
}

}  // namespace kfac
