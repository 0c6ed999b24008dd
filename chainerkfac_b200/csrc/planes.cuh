// Products of matrices that lie in memory as planes of fp16 terms, x 2^s = hi + lo
// (row-major, hi in front of lo), C = A B over many problems in one launch, on
// tcgen05 tensor cores with fp32 accumulators.  An operand gives one term or two;
// with two on both sides C = hi*hi + (hi*lo + lo*hi), the cross terms in an
// accumulator of their own: 22 significant bits.
//
// Tiles of 128 x 128, k-blocks of 64: TMA lays both operands out as the MMAs read
// them, whether k runs along the rows or down the columns of the planes, and fills
// zeros past the edges, so any size goes without a copy.  One CTA an SM walks over
// the tiles: warp 0 issues the loads, warp 1 the MMAs, eight warps take the
// accumulators, which are there twice, out of tensor memory while the MMAs go on in
// the other pair.  The tensor core adds with truncation, so a sum of two-term
// products is cut into segments of 512 k that add up in registers, rounded to
// nearest.
//
// Every barrier wait is bounded; a wait that runs out raises the status word.
#pragma once

#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "gemm_simt.cuh"
#include "tc_common.cuh"

namespace kfac {

// Status word of the bounded waits, one in each source file that has products.
static __device__ int g_plane_status = 0;

constexpr int PL_BM = 128;                   // tile sides
constexpr int PL_BK = 64;                    // k of a stage: 128 bytes of fp16
constexpr int PL_TERM = PL_BM * PL_BK * 2;   // bytes of one term of an operand tile
constexpr int PL_STAGE_BYTES = 12 * PL_TERM; // 192 KB of stages, 2 to 4 terms each
constexpr int PL_STAGES_MAX = 6;
constexpr int PL_SEGMENT = 8;                // k-blocks of an accumulator's sum
constexpr int PL_EPI_WARPS = 8;
constexpr int PL_THREADS = 32 * (2 + PL_EPI_WARPS);
constexpr int PL_PIECE = 4096;               // bytes of a warp's staging
constexpr int PL_SMEM =
    PL_STAGE_BYTES + PL_EPI_WARPS * PL_PIECE + 1024 /* control */ + 1024 /* align */;
constexpr int PL_COLS = 512;                 // tensor memory: 2 x (main, cross)

// A pair of planes.
struct Planes {
  __half* p;
  long long plane;       // elements from hi to lo
  int ld;                // elements of a row, a multiple of 8
};

struct alignas(64) PlaneProblem {
  CUtensorMap ma, mb;
  int M, N, K;
  int tiles_n, tile_begin;
  int lower;             // square and symmetric: tiles on and below the diagonal
  int a_mn, b_mn;        // k runs down the columns of the operand's planes
  int same;              // A and B are the same operand
  int ta, tb;            // terms of the operands, the same sum in all of a launch
  Planes out;            // of the result (not used by every epilogue)
  Planes add;
  float scale;
  void* dst;
  void* param;
};

template <int N>
struct PlaneLaunch {
  PlaneProblem p[N];
  int n;
  int tiles;
  int terms;             // of both operands
};

struct PlaneControl {
  unsigned long long full[PL_STAGES_MAX];
  unsigned long long empty[PL_STAGES_MAX];
  unsigned long long accum[2];
  unsigned long long drained[2];
  unsigned tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(PlaneControl) <= 1024, "control block");

__device__ __forceinline__ void pl_load(unsigned dst, const CUtensorMap* map, int x,
                                        int y, int z, unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// One term of an operand tile: rows r0.. of it, k-block kb.  Rows down the planes: a
// box of 128 rows x 64 k; rows along the planes: two boxes of 64 k x 64 rows.
__device__ __forceinline__ void pl_load_term(unsigned dst, const CUtensorMap* map,
                                             int mn, int r0, int kb, int term,
                                             unsigned long long* bar) {
  if (!mn) {
    pl_load(dst, map, kb * PL_BK, r0, term, bar);
  } else {
    pl_load(dst, map, r0, kb * PL_BK, term, bar);
    pl_load(dst + PL_TERM / 2, map, r0 + 64, kb * PL_BK, term, bar);
  }
}

// 32 columns of this lane's accumulator row.
__device__ __forceinline__ void pl_ld32(unsigned taddr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, "
      "%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
        "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// Two values as fp16 terms, rounded to nearest.  Beyond the range hi is infinite and
// lo not a number: what does not fit shows.
__device__ __forceinline__ void pl_split2(float y0, float y1, unsigned& hi,
                                          unsigned& lo) {
  const __half2 h = __floats2half2_rn(y0, y1);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(y0 - f.x, y1 - f.y);
  hi = *reinterpret_cast<const unsigned*>(&h);
  lo = *reinterpret_cast<const unsigned*>(&l);
}

// What an epilogue's warp has: 64 columns c0.. of 32 rows r0.. (row: the lane), and
// 4 KB of shared memory of its own.
struct PlaneTile {
  int r0, c0, lane;
  unsigned char* piece;
};

// v as planes, rows r0 + lane, and with `mirror` (a tile below the diagonal of a
// symmetric result) its transpose.  Rows go out as 128 (transposed: 64) bytes, turned
// in shared memory.
__device__ __forceinline__ void pl_store_planes(const PlaneTile& t, const Planes& o,
                                                const float (&v)[64], int M, int N,
                                                int terms, bool mirror) {
  unsigned char* const piece = t.piece;
  const int lane = t.lane;
#pragma unroll
  for (int term = 0; term < 2; ++term) {
    if (term >= terms) break;
    __half* const base = o.p + (term ? o.plane : 0);
    unsigned w[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      unsigned hi, lo;
      pl_split2(v[2 * i], v[2 * i + 1], hi, lo);
      w[i] = term ? lo : hi;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<uint4*>(piece + lane * 128 + ((j ^ (lane & 7)) << 4)) =
          make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3), j = lane & 7;
      const uint4 x =
          *reinterpret_cast<const uint4*>(piece + r * 128 + ((j ^ (r & 7)) << 4));
      // (a row's last words may pass its end: the plane has the room)
      if (t.r0 + r < M && t.c0 + 8 * j < N)
        *reinterpret_cast<uint4*>(base + (long long)(t.r0 + r) * o.ld + t.c0 +
                                  8 * j) = x;
    }
    if (!mirror) continue;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      __half* const at = reinterpret_cast<__half*>(piece) + 64 * i + lane;
      const __half2 x = *reinterpret_cast<const __half2*>(&w[i]);
      at[0] = __low2half(x);
      at[32] = __high2half(x);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = 8 * i + (lane >> 2), j = lane & 3;
      const uint4 x = *reinterpret_cast<const uint4*>(piece + c * 64 + 16 * j);
      if (t.c0 + c < N && t.r0 + 8 * j < M)
        *reinterpret_cast<uint4*>(base + (long long)(t.c0 + c) * o.ld + t.r0 +
                                  8 * j) = x;
    }
  }
}

// Which problem a tile belongs to.
template <int N>
__device__ __forceinline__ const PlaneProblem& pl_problem(const PlaneLaunch<N>& l,
                                                          int tile) {
  int f = 0;
  for (int i = 1; i < l.n; ++i)
    if (l.p[i].tile_begin <= tile) f = i;
  return l.p[f];
}

__device__ __forceinline__ void pl_tile_at(const PlaneProblem& g, int tile, int& m0,
                                           int& n0) {
  const int t = tile - g.tile_begin;
  int bi, bj;
  if (g.lower) {
    tri_tile(t, bi, bj);
  } else {
    bi = t / g.tiles_n;
    bj = t - bi * g.tiles_n;
  }
  m0 = bi * PL_BM;
  n0 = bj * PL_BM;
}

// Epi: the epilogue's type; epi.store(problem, tile, v) takes the sums of a warp's
// part of a tile, unscaled.
template <int N, typename Epi>
__global__ void __launch_bounds__(PL_THREADS, 1)
plane_kernel(const __grid_constant__ PlaneLaunch<N> l,
             const __grid_constant__ Epi epi) {
  int* const status = &g_plane_status;
  extern __shared__ unsigned char pl_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(pl_smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* const pieces = smem + PL_STAGE_BYTES;
  PlaneControl* ctl =
      reinterpret_cast<PlaneControl*>(pieces + PL_EPI_WARPS * PL_PIECE);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int stage_bytes = l.terms * PL_TERM;
  const int stages = PL_STAGE_BYTES / stage_bytes;
  const bool cross = l.terms > 2, cut = l.terms == 4;

  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < PL_STAGES_MAX; ++s) {
        mbar_init(&ctl->full[s], 1);
        mbar_init(&ctl->empty[s], 1);
      }
      for (int b = 0; b < 2; ++b) {
        mbar_init(&ctl->accum[b], 1);
        mbar_init(&ctl->drained[b], PL_EPI_WARPS);
      }
      ctl->abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile(
        "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
        ::"r"(smem_u32(&ctl->tmem_base)), "r"(PL_COLS)
        : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;"
                 ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  let_next_launch_begin();
  wait_for_launch_before();

  const unsigned tmem = ctl->tmem_base;
  if (warp == 0) {
    if (elect_one()) {
      // what the launch before wrote is read by the copy engine
      asm volatile("fence.proxy.async;" ::: "memory");
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < l.tiles; tile += gridDim.x) {
        const PlaneProblem& g = pl_problem(l, tile);
        int m0, n0;
        pl_tile_at(g, tile, m0, n0);
        const bool share = g.same && m0 == n0;
        const int nkb = (g.K + PL_BK - 1) / PL_BK, ta = g.ta, tb = g.tb;
        const unsigned bytes = (share ? ta : ta + tb) * PL_TERM;
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = it % stages;
          if (it >= stages &&
              !mbar_wait_status(&ctl->empty[s], ((it / stages) - 1) & 1,
                                &ctl->abort_flag, status)) {
            ok = false;
            break;
          }
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                       ::"r"(smem_u32(&ctl->full[s])), "r"(bytes)
                       : "memory");
          const unsigned st = smem_u32(smem + s * stage_bytes);
          for (int t = 0; t < ta; ++t)
            pl_load_term(st + t * PL_TERM, &g.ma, g.a_mn, m0, kb, t, &ctl->full[s]);
          if (share) continue;
          for (int t = 0; t < tb; ++t)
            pl_load_term(st + (ta + t) * PL_TERM, &g.mb, g.b_mn, n0, kb, t,
                         &ctl->full[s]);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      int it = 0, seg = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < l.tiles; tile += gridDim.x) {
        const PlaneProblem& g = pl_problem(l, tile);
        int m0, n0;
        pl_tile_at(g, tile, m0, n0);
        const bool share = g.same && m0 == n0;
        const int nkb = (g.K + PL_BK - 1) / PL_BK, ta = g.ta, tb = g.tb;
        const bool amn = g.a_mn, bmn = g.b_mn;
        const unsigned idesc = tc_half_desc(PL_BM, amn, bmn);
        // from 16 k to the next (16-byte units)
        const unsigned long long adv_a = (amn ? 2048 : 32) >> 4;
        const unsigned long long adv_b = (bmn ? 2048 : 32) >> 4;
        unsigned d = 0;
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = it % stages;
          const bool fresh = kb == 0 || (cut && kb % PL_SEGMENT == 0);
          if (fresh) {
            const int b = seg & 1;
            d = tmem + b * (PL_COLS / 2);
            if (seg >= 2 &&
                !mbar_wait_status(&ctl->drained[b], ((seg >> 1) - 1) & 1,
                                  &ctl->abort_flag, status)) {
              ok = false;
              break;
            }
          }
          if (!mbar_wait_status(&ctl->full[s], (it / stages) & 1, &ctl->abort_flag,
                                status)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned sa = smem_u32(smem + s * stage_bytes);
          const unsigned sb = share ? sa : sa + ta * PL_TERM;
          unsigned long long a =
              amn ? tc_smem_desc_mn(sa, PL_TERM / 2) : tc_smem_desc(sa);
          unsigned long long b =
              bmn ? tc_smem_desc_mn(sb, PL_TERM / 2) : tc_smem_desc(sb);
          const unsigned long long lo = PL_TERM >> 4;
#pragma unroll
          for (int kk = 0; kk < PL_BK / 16; ++kk, a += adv_a, b += adv_b) {
            const unsigned acc = !fresh || kk != 0;
            if (tb == 2) tc_mma_half(d + PL_BM, a, b + lo, idesc, acc);
            if (ta == 2) tc_mma_half(d + PL_BM, a + lo, b, idesc, acc | (tb == 2));
            tc_mma_half(d, a, b, idesc, acc);
          }
          tc_commit(&ctl->empty[s]);
          if (kb + 1 == nkb || (cut && (kb + 1) % PL_SEGMENT == 0)) {
            tc_commit(&ctl->accum[seg & 1]);
            ++seg;
          }
        }
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, h = (warp - 2) >> 2;
    PlaneTile t;
    t.lane = lane;
    t.piece = pieces + (warp - 2) * PL_PIECE;
    int seg = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < l.tiles; tile += gridDim.x) {
      const PlaneProblem& g = pl_problem(l, tile);
      int m0, n0;
      pl_tile_at(g, tile, m0, n0);
      t.r0 = m0 + 32 * q;
      t.c0 = n0 + 64 * h;
      const int nkb = (g.K + PL_BK - 1) / PL_BK;
      const int nseg = cut ? (nkb + PL_SEGMENT - 1) / PL_SEGMENT : 1;
      float v[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) v[i] = 0.f;
#pragma unroll 1
      for (int k = 0; k < nseg; ++k, ++seg) {
        const int b = seg & 1;
        ok = mbar_wait_status(&ctl->accum[b], (seg >> 1) & 1, &ctl->abort_flag,
                              status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned at = tmem + ((unsigned)(32 * q) << 16) + b * (PL_COLS / 2) +
                            64 * h;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          unsigned x[32], y[32];
          pl_ld32(at + 32 * half, x);
          if (cross) pl_ld32(at + PL_BM + 32 * half, y);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float sum = __uint_as_float(x[i]);
            if (cross) sum += __uint_as_float(y[i]);
            v[32 * half + i] += sum;
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->drained[b]);
      }
      if (!ok) break;
      if (t.r0 < g.M && t.c0 < g.N)
        epi.store(g, t, v, g.lower && m0 != n0);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) tc_release(tmem, PL_COLS, ctl->abort_flag != 0);
}

// ----------------------------------------------------------------- host side
typedef CUresult (*PlaneEncodeFn)(
    CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// (through the runtime's driver entry point: the library must load on machines
// without a driver)
inline int plane_encode_fn(PlaneEncodeFn* out) {
  static PlaneEncodeFn fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    KFAC_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault,
                                      &q));
    KFAC_REQUIRE(q == cudaDriverEntryPointSuccess && p != nullptr,
                 "the driver has no cuTensorMapEncodeTiled");
    fn = reinterpret_cast<PlaneEncodeFn>(p);
  }
  *out = fn;
  return KFAC_OK;
}

// Tensor map of rows x cols planes: boxes of 64 columns and 128 rows (k along the
// rows) or 64 (`mn`: k down the columns) of one plane.  Past the edges: zeros.
inline int plane_map(CUtensorMap* map, const Planes& o, int rows, int cols, bool mn) {
  PlaneEncodeFn encode = nullptr;
  const int rc = plane_encode_fn(&encode);
  if (rc != KFAC_OK) return rc;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 2};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)o.plane * 2};
  const cuuint32_t box[3] = {64, mn ? 64u : 128u, 1};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = encode(
      map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, o.p, dims, strides, box, es,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(KFAC_ERR_CUDA,
                "cuTensorMapEncodeTiled failed (%d) for planes of %d x %d", (int)r,
                rows, cols);
  return KFAC_OK;
}

// Numbers the tiles of l.p[0 .. l.n).
template <int N>
void plane_number_tiles(PlaneLaunch<N>& l) {
  int total = 0;
  for (int i = 0; i < l.n; ++i) {
    PlaneProblem& g = l.p[i];
    const int tm = (g.M + PL_BM - 1) / PL_BM, tn = (g.N + PL_BM - 1) / PL_BM;
    g.tiles_n = tn;
    g.tile_begin = total;
    total += g.lower ? tm * (tm + 1) / 2 : tm * tn;
  }
  l.tiles = total;
  l.terms = l.n > 0 ? l.p[0].ta + l.p[0].tb : 0;
}

template <int N, typename Epi>
int plane_launch(const char* name, const PlaneLaunch<N>& l, const Epi& epi,
                 bool early, cudaStream_t stream) {
  if (l.tiles == 0) return KFAC_OK;
  static std::mutex mu;
  static bool done[64] = {false};
  int dev = 0;
  KFAC_CUDA(cudaGetDevice(&dev));
  KFAC_REQUIRE(dev >= 0 && dev < 64, "device index %d unsupported", dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      KFAC_CUDA(cudaFuncSetAttribute(plane_kernel<N, Epi>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     PL_SMEM));
      done[dev] = true;
    }
  }
  return launch_behind(name, early, plane_kernel<N, Epi>,
                       std::min(l.tiles, sm_count()), PL_THREADS, PL_SMEM, stream, l,
                       epi);
}

}  // namespace kfac
