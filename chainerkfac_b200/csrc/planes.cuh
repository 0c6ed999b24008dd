// Products of matrices that lie in memory as planes of fp16 terms, x 2^s = hi + lo
// (row-major, hi in front of lo), C = A B over many problems in one launch, on
// tcgen05 tensor cores with fp32 accumulators: C = (hi*lo + lo*hi) + hi*hi in one
// accumulator, 22 significant bits of every operand.
//
// Tiles of 256 x 256 by pairs of CTAs (cta_group::2: each holds 128 rows of A and of
// C, and half of B's rows), or of 128 x 128 by one CTA where there are few of them,
// k-blocks of 64: TMA lays both operands out as the MMAs read them, whether k runs
// along the rows or down the columns of the planes, and fills zeros past the edges, so
// any size goes without a copy.  In each CTA warp 0 issues the loads and, in the first
// of a pair, warp 1 the MMAs; eight warps take the accumulators, which are there twice,
// out of tensor memory while the MMAs go on in the other one.
//
// The tensor core adds with truncation, so a long sum comes out too small by what
// its number of additions makes: a sum is cut every two k-blocks (or each) and
// the segments are added in registers, rounded to nearest; within a k-block the cross
// terms, 2^-11 of the others, go first, when the accumulator is small.
//
// Launches with fewer tiles than the GPU has room for share the sum of a tile among
// up to eight pairs (four CTAs) of a cluster, which hand each other their parts through
// distributed shared memory, added in the order of k.
//
// Every barrier wait is bounded; a wait that runs out raises the status word.
#pragma once

#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "gemm_simt.cuh"
#include "tc_common.cuh"

namespace kfac {

// Status word of the bounded waits, one in each source file that has products.
static __device__ int g_plane_status = 0;

constexpr int PL_ROWS = 128;                 // rows of a CTA's part of A, B and C
constexpr int PL_BK = 64;                    // k of a stage: 128 bytes of fp16
constexpr int PL_TERM = PL_ROWS * PL_BK * 2; // bytes of one term of such a part
constexpr int PL_STAGE = 4 * PL_TERM;        // bytes of a stage: two terms of A and of B
constexpr int PL_STAGES = 3;
constexpr int PL_STAGE_BYTES = PL_STAGES * PL_STAGE;
// k-blocks of an accumulator's sum.  4096 x 4096, five steps: 4.3 ms and an error of
// 1.0e-6 with one, 3.5 ms and 1.9e-6 with two, 3.4 ms and 3.7e-6 with four: of one, a
// segment is in the tensor cores for less time than it takes to read.  Small tiles'
// short sums are read in no more time than what is around them: of up to PL_SHORT
// k-blocks, one (300 x 1000 1.9e-6 and 3.7e-6, both 140 us; of any length 1000 x 1000
// 253 us and 228, 512 x 4608 237 and 204).
constexpr int PL_SHORT = 6;
constexpr int PL_EPI_WARPS = 8;
constexpr int PL_THREADS = 32 * (4 + PL_EPI_WARPS);
constexpr int PL_PIECE = 4096;               // bytes of a warp's staging
constexpr int PL_SMEM =
    PL_STAGE_BYTES + PL_EPI_WARPS * PL_PIECE + 1024 /* control */ + 1024 /* align */;
constexpr int PL_COLS = 512;                 // tensor memory: two accumulators
// Cycles that a small tile takes beside its k-blocks with a shared sum and without
// (plane_split).
constexpr double PL_SMALL_SHARE = 5000, PL_SMALL_END = 5000;
static_assert(256 * 512 <= PL_STAGE_BYTES, "parts of a shared sum");

// A pair of planes.
struct Planes {
  __half* p;
  long long plane;       // elements from hi to lo
  int ld;                // elements of a row, a multiple of 8
};

// What the warps of a launch read of a problem, copied to registers for a tile.
struct PlaneFields {
  int M, N, K;
  int tiles_n, tile_begin;
  int lower;             // square and symmetric: tiles on and below the diagonal
  int a_mn, b_mn;        // k runs down the columns of the operand's planes
  int same;              // A and B are the same operand
  int odd;               // k-blocks of an accumulator's sum, less one: 0 or 1 (PL_SHORT)
  Planes out;            // of the result (not used by every epilogue)
  Planes add;
  float scale;
  float gain;            // makes up for what the sums lose (plane_gain)
  void* dst;
  void* param;
};

struct alignas(64) PlaneProblem {
  CUtensorMap ma, mb;
  PlaneFields f;
};

template <int N>
struct PlaneLaunch {
  PlaneProblem p[N];
  int n;
  int tiles;
  int split;             // CTAs, or pairs of them, that share a tile
  const int* rows;       // the rows of a launch's only problem, where the device counts
                         // them (M is then the most there can be); or null
};

struct PlaneControl {
  unsigned long long full[PL_STAGES];
  unsigned long long empty[PL_STAGES];
  unsigned long long accum[2];
  unsigned long long drained[2];
  unsigned tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(PlaneControl) <= 1024, "control block");

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// All threads of the cluster; what was written before is seen behind it.
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same place in another CTA's shared memory.
__device__ __forceinline__ unsigned cluster_addr(unsigned addr, unsigned rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_arrive(unsigned bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];"
               ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void cluster_store(unsigned addr, float a, float b, float c,
                                              float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a),
               "f"(b), "f"(c), "f"(d)
               : "memory");
}

// D = f32, A = B = f16, M = N = 128 by one CTA, 256 by two.
template <int G>
__device__ __forceinline__ unsigned pl_desc(bool a_mn, bool b_mn) {
  return (1u << 4) | ((unsigned)a_mn << 15) | ((unsigned)b_mn << 16) |
         ((unsigned)(128 * G >> 3) << 17) | ((unsigned)(128 * G >> 4) << 24);
}
template <int G>
__device__ __forceinline__ void pl_mma(unsigned tmem_d, unsigned long long da,
                                       unsigned long long db, unsigned idesc,
                                       unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::%5.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "n"(G)
      : "memory");
}
// Arrives at the barrier in both CTAs of the pair (`mask`) once the MMAs are done.
template <int G>
__device__ __forceinline__ void pl_commit(unsigned long long* bar,
                                          unsigned short mask) {
  if (G == 1) {
    tc_commit(bar);
    return;
  }
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster."
      "multicast::cluster.b64 [%0], %1;"
      ::"r"(smem_u32(bar)), "h"(mask)
      : "memory");
}

// G: CTAs of a tile.  Of a pair both count at the first one's barrier.
template <int G>
__device__ __forceinline__ void pl_load(unsigned dst, const CUtensorMap* map, int x,
                                        int y, int z, unsigned bar) {
  if (G == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
        "complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
    return;
  }
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Both terms of an operand tile from (x, y) of its planes.  Rows down the planes: a box
// of 128 rows x 64 k; rows along them (`mn`): two boxes of 64 k x 64 rows.
template <int G>
__device__ __forceinline__ void pl_load_terms(unsigned dst, const CUtensorMap* map,
                                              bool mn, int x, int y, unsigned bar) {
  pl_load<G>(dst, map, x, y, 0, bar);
  if (mn) pl_load<G>(dst + PL_TERM / 2, map, x + 64, y, 0, bar);
  pl_load<G>(dst + PL_TERM, map, x, y, 1, bar);
  if (mn) pl_load<G>(dst + PL_TERM + PL_TERM / 2, map, x + 64, y, 1, bar);
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

// What an epilogue gets at a time: 32 rows from r0 and 32 columns from c0, and 4 KB of
// shared memory of the warp's own.  v[16 f + 4 j + 2 h + e] is row 16 f + 8 h +
// lane / 4, column 8 j + 2 (lane % 4) + e: what the matrix stores and loads of shared
// memory have in a register.
struct PlaneTile {
  int r0, c0, lane;
  unsigned char* piece;
};

__device__ __forceinline__ void st_matrix(unsigned addr, unsigned a, unsigned b,
                                          unsigned c, unsigned d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};"
               ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void st_matrix_t(unsigned addr, unsigned a, unsigned b,
                                            unsigned c, unsigned d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
               ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void ld_matrix(unsigned addr, unsigned& a, unsigned& b,
                                          unsigned& c, unsigned& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}

// For epilogues with nothing to do ahead.
struct NothingAhead {};

// 32 rows of 64 bytes in shared memory, without bank conflicts: 16-byte word j of a row.
__device__ __forceinline__ int row64_off(int row, int j) {
  return row * 64 + ((j ^ ((row >> 1) & 3)) << 4);
}

// A tile's 16-bit pairs (w[8 f + 2 j + h], one word per row and column pair) from the
// registers to rows of 64 bytes, or transposed.
__device__ __forceinline__ void pl_put_pairs(unsigned piece, const unsigned (&w)[16],
                                             int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    st_matrix(piece + row64_off(lane, j), w[2 * j], w[2 * j + 1], w[8 + 2 * j],
              w[8 + 2 * j + 1]);
}
__device__ __forceinline__ void pl_put_pairs_t(unsigned piece, const unsigned (&w)[16],
                                               int lane) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {            // eight rows: 16-byte word g of a column
    const int at = 8 * (g >> 1) + (g & 1);
    st_matrix_t(piece + row64_off(lane, g), w[at], w[at + 2], w[at + 4], w[at + 6]);
  }
}

// Those rows to memory, 16 bytes a lane: row r0 + r of `rows`, columns from c0 of
// `cols` (a row's last word may pass its end: the plane has the room).
__device__ __forceinline__ void pl_rows_out(unsigned piece, __half* base, int ld,
                                            int r0, int rows, int c0, int cols,
                                            int lane) {
  const int j = lane & 3, r = lane >> 2;
  __half* to = base + (long long)(r0 + r) * ld + c0 + 8 * j;
  const unsigned from = piece + row64_off(r, j);   // (eight rows on: the same turn)
  const int left = c0 + 8 * j < cols ? rows - r0 - r : 0;
  const long long step = 8LL * ld;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(from + 512 * i)
                 : "memory");
    if (8 * i < left) *reinterpret_cast<uint4*>(to) = x;
    to += step;
  }
}

// v as planes, and with `mirror` (below the diagonal of a symmetric result) its
// transpose.
__device__ __forceinline__ void pl_store_planes(const PlaneTile& t, const Planes& o,
                                                const float (&v)[32], int M, int N,
                                                bool mirror) {
  const unsigned piece = smem_u32(t.piece);
  unsigned hi[16], lo[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) pl_split2(v[2 * i], v[2 * i + 1], hi[i], lo[i]);
#pragma unroll 1
  for (int term = 0; term < 2; ++term) {
    __half* const base = o.p + (term ? o.plane : 0);
    __syncwarp();
    pl_put_pairs(piece, hi, t.lane);
    if (mirror) pl_put_pairs_t(piece + 2048, hi, t.lane);
    __syncwarp();
    pl_rows_out(piece, base, o.ld, t.r0, M, t.c0, N, t.lane);
    if (mirror) pl_rows_out(piece + 2048, base, o.ld, t.c0, N, t.r0, M, t.lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) hi[i] = lo[i];
  }
}

// 32 x 32 values as rows of 128 bytes in shared memory, 16-byte words turned by the row
// (no bank conflicts): what a lane reads back is a column, or a word, of a row.
__device__ __forceinline__ unsigned row128_at(unsigned piece, int row, int word) {
  return piece + row * 128 + ((word ^ (row & 7)) << 4);
}
__device__ __forceinline__ void pl_put_floats(unsigned piece, const float (&v)[32],
                                              int lane) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const int row = 16 * (i >> 4) + 8 * ((i >> 1) & 1) + (lane >> 2);
    asm volatile("st.shared.v2.f32 [%0], {%1, %2};"
                 ::"r"(row128_at(piece, row, 2 * ((i >> 2) & 3) + ((lane & 3) >> 1)) +
                       8 * (lane & 1)),
                   "f"(v[i]), "f"(v[i + 1])
                 : "memory");
  }
}
__device__ __forceinline__ float4 pl_word(unsigned piece, int row, int word) {
  float4 x;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(row128_at(piece, row, word))
               : "memory");
  return x;
}
__device__ __forceinline__ float pl_float(unsigned piece, int row, int col) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];"
               : "=f"(x)
               : "r"(row128_at(piece, row, col >> 2) + 4 * (col & 3))
               : "memory");
  return x;
}

// Which problem a tile belongs to.
template <int N>
__device__ __forceinline__ const PlaneProblem& pl_problem(const PlaneLaunch<N>& l,
                                                          int tile) {
  int f = 0;
  for (int i = 1; i < l.n; ++i)
    if (l.p[i].f.tile_begin <= tile) f = i;
  return l.p[f];
}

template <int G>
__device__ __forceinline__ void pl_tile_at(const PlaneFields& g, int tile, int& m0,
                                           int& n0) {
  const int t = tile - g.tile_begin;
  int bi, bj;
  if (g.lower) {
    tri_tile(t, bi, bj);
  } else {
    bi = t / g.tiles_n;
    bj = t - bi * g.tiles_n;
  }
  m0 = bi * 128 * G;
  n0 = bj * 128 * G;
}

// Epi: the epilogue's type.  epi.begin(problem, tile) is called for a warp's rows and
// its first columns before the sums are there; epi.store(problem, tile, v, mirror,
// what begin gave) takes the sums of a PlaneTile, unscaled.
// G: CTAs of a tile.
template <int N, typename Epi, int G>
__global__ void __launch_bounds__(PL_THREADS, 1)
plane_kernel(const __grid_constant__ PlaneLaunch<N> l,
             const __grid_constant__ Epi epi) {
  constexpr int TILE = 128 * G;            // sides
  constexpr int COLS = TILE / 2;           // columns of an epilogue's warp
  constexpr int BUFFER = PL_COLS / 2;      // tensor memory of an accumulator
  int* const status = &g_plane_status;
  extern __shared__ unsigned char pl_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(pl_smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* const pieces = smem + PL_STAGE_BYTES;
  PlaneControl* ctl =
      reinterpret_cast<PlaneControl*>(pieces + PL_EPI_WARPS * PL_PIECE);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = l.split;
  const unsigned rank = cluster_rank(), side = rank % G, first = rank - side;
  const int part = (int)(rank / G);                // of a shared sum
  const int tile0 = blockIdx.x / (G * S), step = gridDim.x / (G * S);

  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < PL_STAGES; ++s) {
        mbar_init(&ctl->full[s], 1);
        mbar_init(&ctl->empty[s], 1);
      }
      for (int b = 0; b < 2; ++b) {
        mbar_init(&ctl->accum[b], 1);
        mbar_init(&ctl->drained[b], G * PL_EPI_WARPS);
      }
      ctl->abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile(
        "tcgen05.alloc.cta_group::%2.sync.aligned.shared::cta.b32 [%0], %1;"
        ::"r"(smem_u32(&ctl->tmem_base)), "r"(PL_COLS), "n"(G)
        : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::%0.sync.aligned;"
                 ::"n"(G)
                 : "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  let_next_launch_begin();
  // (each role waits for the launch before where it first reads or writes memory)

  const unsigned tmem = ctl->tmem_base;
  // Parts of a shared sum go to the end of the stages; where no k-block of the tile lies
  // there, nobody has to wait for the others' MMAs before writing them.
  constexpr int PARTS = TILE * 512;
  bool apart = true;
  if (S > 1) {
    const PlaneFields& g = pl_problem(l, tile0).f;
    const int all = (g.K + PL_BK - 1) / PL_BK;
    apart = (all + S - 1) / S * PL_STAGE <= PL_STAGE_BYTES - PARTS;
  }
  // k-blocks of a tile that this pair adds up
  auto range = [&](const PlaneFields& g, int& kb0, int& nkb) {
    const int all = (g.K + PL_BK - 1) / PL_BK, each = (all + S - 1) / S;
    kb0 = min(part * each, all);
    nkb = min(each, all - kb0);
  };
  int tiles = l.tiles, counted = 0;
  if (l.rows != nullptr) {
    wait_for_launch_before();
    counted = *reinterpret_cast<const volatile int*>(l.rows);
    tiles = (counted + TILE - 1) / TILE * l.p[0].f.tiles_n;
  }
  // (The loops over k-blocks carry stages, phases, coordinates and descriptors along:
  // with divisions and addresses made anew each of the two threads took 500 cycles and
  // more for one, waits aside.)
  if (warp == 0) {
    if (elect_one()) {
      int s = 0;
      unsigned turn = 1;                     // (the first round finds all stages empty)
      bool ok = true, begun = false;
      // both CTAs' loads count at the first one's barrier
      const unsigned own = smem_u32(ctl->full), bars = cluster_addr(own, first);
      const unsigned stage0 = smem_u32(smem);
      for (int tile = tile0; ok && tile < tiles; tile += step) {
        const PlaneProblem& p = pl_problem(l, tile);
        const PlaneFields g = p.f;
        int m0, n0, kb0, nkb;
        pl_tile_at<G>(g, tile, m0, n0);
        range(g, kb0, nkb);
        const bool share = g.same && m0 == n0, amn = g.a_mn, bmn = g.b_mn;
        const unsigned bytes = G * (share ? 2 : 4) * PL_TERM;
        const int ra = m0 + PL_ROWS * side, rb = n0 + PL_ROWS * side;
        int k = kb0 * PL_BK;
        if (!begun) {
          begun = true;
          asm volatile("prefetch.tensormap [%0];" ::"l"(&p.ma) : "memory");
          asm volatile("prefetch.tensormap [%0];" ::"l"(&p.mb) : "memory");
          wait_for_launch_before();
          // what it wrote is read by the copy engine
          asm volatile("fence.proxy.async.global;" ::: "memory");
        }
        for (int kb = 0; kb < nkb; ++kb, k += PL_BK) {
          if (!mbar_wait_status(&ctl->empty[s], turn, &ctl->abort_flag, status)) {
            ok = false;
            break;
          }
          const unsigned bar = bars + 8 * s, st = stage0 + s * PL_STAGE;
          if (side == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                         ::"r"(own + 8 * s), "r"(bytes)
                         : "memory");
          pl_load_terms<G>(st, &p.ma, amn, amn ? ra : k, amn ? k : ra, bar);
          if (!share)
            pl_load_terms<G>(st + 2 * PL_TERM, &p.mb, bmn, bmn ? rb : k, bmn ? k : rb,
                             bar);
          if (++s == PL_STAGES) {
            s = 0;
            turn ^= 1;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // (not before there is something to multiply: the waits are bounded)
    wait_for_launch_before();
    if (side == 0 && elect_one()) {
      const unsigned short both = (unsigned short)(3u << first);
      int s = 0, seg = 0;
      unsigned turn = 0;
      bool ok = true;
      const unsigned stage0 = smem_u32(smem);
      for (int tile = tile0; ok && tile < tiles; tile += step) {
        const PlaneFields g = pl_problem(l, tile).f;
        int m0, n0, kb0, nkb;
        pl_tile_at<G>(g, tile, m0, n0);
        range(g, kb0, nkb);
        const int odd = g.odd;
        const bool share = g.same && m0 == n0;
        const bool amn = g.a_mn, bmn = g.b_mn;
        const unsigned idesc = pl_desc<G>(amn, bmn);
        // from 16 k to the next (16-byte units)
        const unsigned long long adv_a = (amn ? 2048 : 32) >> 4;
        const unsigned long long adv_b = (bmn ? 2048 : 32) >> 4;
        const unsigned long long lo = PL_TERM >> 4;
        const unsigned stage_b = share ? stage0 : stage0 + 2 * PL_TERM;
        const unsigned long long a0 =
            amn ? tc_smem_desc_mn(stage0, PL_TERM / 2) : tc_smem_desc(stage0);
        const unsigned long long b0 =
            bmn ? tc_smem_desc_mn(stage_b, PL_TERM / 2) : tc_smem_desc(stage_b);
        unsigned d = 0;
        for (int kb = 0; kb < nkb; ++kb) {
          const bool fresh = (kb & odd) == 0;
          if (fresh) {
            const int b = seg & 1;
            d = tmem + b * BUFFER;
            if (seg >= 2 &&
                !mbar_wait_status(&ctl->drained[b], ((seg >> 1) - 1) & 1,
                                  &ctl->abort_flag, status)) {
              ok = false;
              break;
            }
          }
          if (!mbar_wait_status(&ctl->full[s], turn, &ctl->abort_flag, status)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned long long at = (unsigned)(s * PL_STAGE) >> 4;
          const unsigned long long a = a0 + at, b = b0 + at;
          unsigned acc = !fresh;
#pragma unroll
          for (int kk = 0; kk < PL_BK / 16; ++kk) {
            pl_mma<G>(d, a + kk * adv_a, b + lo + kk * adv_b, idesc, acc);
            acc = 1;
          }
#pragma unroll
          for (int kk = 0; kk < PL_BK / 16; ++kk)
            pl_mma<G>(d, a + lo + kk * adv_a, b + kk * adv_b, idesc, 1);
#pragma unroll
          for (int kk = 0; kk < PL_BK / 16; ++kk)
            pl_mma<G>(d, a + kk * adv_a, b + kk * adv_b, idesc, 1);
          pl_commit<G>(&ctl->empty[s], both);
          if (kb + 1 == nkb || (kb & odd) == odd) {
            pl_commit<G>(&ctl->accum[seg & 1], both);
            ++seg;
          }
          if (++s == PL_STAGES) {
            s = 0;
            turn ^= 1;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int q = warp & 3, h = (warp >> 2) - 1;
    PlaneTile t;
    t.lane = lane;
    t.piece = pieces + (warp - 4) * PL_PIECE;
    int seg = 0;
    bool ok = true;
    wait_for_launch_before();
    for (int tile = tile0; ok && tile < tiles; tile += step) {
      PlaneFields g = pl_problem(l, tile).f;
      if (l.rows != nullptr) g.M = counted;
      int m0, n0, kb0, nkb;
      pl_tile_at<G>(g, tile, m0, n0);
      range(g, kb0, nkb);
      t.r0 = m0 + PL_ROWS * side + 32 * q;
      const bool mirror = g.lower && m0 != n0;
      const int nseg = (nkb + g.odd) >> g.odd;
      t.c0 = n0 + COLS * h;
      const auto ahead = epi.begin(g, t);
      float v[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) v[i] = 0.f;
#pragma unroll 1
      for (int k = 0; k < nseg; ++k, ++seg) {
        const int b = seg & 1;
        ok = mbar_wait_status(&ctl->accum[b], (seg >> 1) & 1, &ctl->abort_flag,
                              status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned at = tmem + ((unsigned)(32 * q) << 16) + b * BUFFER + COLS * h;
#pragma unroll
        for (int u = 0; u < COLS / 32; ++u) {
          float x[16], y[16];
          tc_ld_16x32(at + 32 * u, x);
          tc_ld_16x32(at + (16u << 16) + 32 * u, y);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[32 * u + i] += x[i];
            v[32 * u + 16 + i] += y[i];
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0)
          cluster_arrive(cluster_addr(smem_u32(&ctl->drained[b]), first));
      }
      if (S > 1) {
        // A shared sum (the cluster's only tile): the pairs own a part of the columns
        // each, a multiple of the 32 that 32 registers hold.  Parts lie by pair, rows'
        // quarter, four registers, lane.
        const int width = TILE / S, groups = width / 4;
        unsigned char* const parts = smem + PL_STAGE_BYTES - PARTS;
        const unsigned base = smem_u32(parts);
        if (!apart) cluster_sync();          // the MMAs have read all stages
        if (ok) {
#pragma unroll
          for (int i = 0; i < COLS / 4; ++i) {
            const int col = COLS * h + 4 * i, owner = col / width;
            const unsigned at =
                base + ((part * 4 + q) * groups + (col - owner * width) / 4) * 512 +
                lane * 16;
            if (owner == part)
              sts128(at, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2],
                                     v[4 * i + 3]));
            else
              cluster_store(cluster_addr(at, G * owner + side), v[4 * i], v[4 * i + 1],
                            v[4 * i + 2], v[4 * i + 3]);
          }
        }
        cluster_sync();
        if (!ok) break;
        // (of 32 columns in all the second half of the warps has none)
        const int mine = max(32, width / 2);
#pragma unroll 1
        for (int c0 = h * mine; c0 < min((h + 1) * mine, width); c0 += 32) {
          float x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0.f;
#pragma unroll 1
          for (int p = 0; p < S; ++p) {
            const unsigned char* from =
                parts + ((p * 4 + q) * groups + c0 / 4) * 512 + lane * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 w = *reinterpret_cast<const float4*>(from + 512 * i);
              x[4 * i] += w.x;
              x[4 * i + 1] += w.y;
              x[4 * i + 2] += w.z;
              x[4 * i + 3] += w.w;
            }
          }
          t.c0 = n0 + part * width + c0;
          if (t.r0 < g.M && t.c0 < g.N) epi.store(g, t, x, mirror, ahead);
        }
        break;
      }
      if (!ok) break;
#pragma unroll
      for (int u = 0; u < COLS / 32; ++u) {
        t.c0 = n0 + COLS * h + 32 * u;
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = v[32 * u + i];
        if (t.r0 < g.M && t.c0 < g.N) epi.store(g, t, x, mirror, ahead);
      }
    }
  }
  if (S > 1 && warp < 4) {
    if (!apart) cluster_sync();
    cluster_sync();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // (nobody leaves while the other may still arrive at its barriers)
  if (G == 2) cluster_sync();
  using Columns = typename std::conditional<G == 2, PairColumns, unsigned>::type;
  if (warp == 1) tc_release(tmem, Columns{PL_COLS}, ctl->abort_flag != 0);
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

// What truncation takes from a segment's sum on average, made good.  An addition
// loses half a unit in the last place of the sum so far, 2^-24 / m of it with a
// mantissa m that is log-uniform: 0.72 2^-24.  Of a sum that grows evenly (a diagonal;
// on average over the places where its large term may stand, any other) the blocks'
// cross terms, 8 additions, meet 0, 1 / n, 2 / n .. of the segment's n blocks' sum, and
// the 4 n others 1 / 4n, 2 / 4n .. 1: 6 n - 3.5 whole ones.  Errors of orthogonalised
// 4096 x 4096 and 1024 x 4096 against fp64, with and without:
// 1.9e-6 and 3.0e-6, 2.3e-6 and 4.0e-6 (fp32 products: 4.3e-6, 3.7e-6).
// (Parts of a shared sum may be shorter than a segment, and a last one always may.)
inline float plane_gain(int all, int each, int segment) {
  float lost = 0.f;
  for (int left = all; left > 0; left -= each)
    for (int part = std::min(left, each); part > 0; part -= segment) {
      const int n = std::min(part, segment);
      lost += n * (6 * n - 3.5f);
    }
  return 1.f + lost / all * 0.72f * exp2f(-24);
}

// Numbers the tiles of l.p[0 .. l.n), of G blocks each.
template <int N>
void plane_number_tiles(PlaneLaunch<N>& l, int G) {
  int total = 0;
  const int side = 128 * G;
  for (int i = 0; i < l.n; ++i) {
    PlaneFields& g = l.p[i].f;
    const int tm = (g.M + side - 1) / side, tn = (g.N + side - 1) / side;
    g.tiles_n = tn;
    g.tile_begin = total;
    total += g.lower ? tm * (tm + 1) / 2 : tm * tn;
  }
  l.tiles = total;
}

// Small tiles or large ones, and how many blocks or pairs share one: what a count of
// cycles comes out least for, with `room[i]` clusters of 2^i of them on the GPU at a
// time.  A k-block of large tiles takes three MMAs of 128 cycles and a little for each
// 16 k.  Small tiles are bound by their shared memory, 128 bytes a cycle: 128 cycles for
// each of four terms that are copied in and 256 for each of three products that read
// two, 1280 (1150 to 1480 were measured; counted as 1040, which fits sums of a few
// k-blocks that begin and end, and leaves long ones to small tiles too often).  Their
// start and end take 7000 cycles (beside the next one's MMAs 2000), a shared sum 5000
// and 500 for each that shares; large ones' 15000, with a symmetric result, which is
// stored twice, 19000, a shared sum no less.  Five steps, us so, with large tiles only,
// with small ones only: 256 x 512 119, 184, 119; 1000 x 1000 228, 269, 228; 512 x 4608
// 202, 281, 202; 3000 x 1000 365, 347, 404; 2048 x 2048 539, 668, 560; 4096 x 4096 3750,
// 3720, 4610; one matrix of each kind of ResNet-50 435, 509, 433; all 54 of it 1225,
// 1305, 1239.  (1000 x 8000, 635, is the furthest behind: 580 with large ones only.)
struct PlaneShape {
  int G, split;
  double cycles;
};
template <int N>
void plane_split(const PlaneLaunch<N>& l, int G, const int* room, PlaneShape& best) {
  const double cycles = G == 2 ? 1584 : 1040;          // of a k-block
  const double end = l.p[0].f.lower ? 17000 : 13000;
  for (int i = 0, s = 1; i < 4 && s <= (G == 2 ? 8 : 4); ++i, s *= 2) {
    if (room[i] <= 0) break;
    const double more = s > 1 ? (G == 2 ? end : PL_SMALL_SHARE) + 500 * s : 2000;
    double longest = 0, sum = 0;
    for (int k = 0; k < l.n; ++k) {
      const int end = k + 1 < l.n ? l.p[k + 1].f.tile_begin : l.tiles;
      const int kb = (l.p[k].f.K + PL_BK - 1) / PL_BK;
      const double one = (kb + s - 1) / s * cycles + more;
      longest = std::max(longest, one);
      sum += one * (end - l.p[k].f.tile_begin);
    }
    // (tiles of one size run in whole waves, of different sizes closer together)
    const double waves = (double)l.tiles / room[i];
    const double busy = l.n == 1 ? sum / l.tiles * std::ceil(waves)
                                 : sum / l.tiles * waves + longest / 2;
    const double time =
        std::max(longest, busy) + (s > 1 ? 0 : G == 2 ? end : PL_SMALL_END);
    if (best.G == 0 || time < best.cycles) best = {G, s, time};
  }
}

// Clusters of G blocks times 1, 2, 4 and 8 that the device has room for.
template <int N, typename Epi, int G>
int plane_prepare(const char* name, int* room) {
  KFAC_CUDA(cudaFuncSetAttribute(plane_kernel<N, Epi, G>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, PL_SMEM));
  KFAC_CUDA(cudaFuncSetAttribute(plane_kernel<N, Epi, G>,
                                 cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(PL_THREADS);
  cfg.dynamicSmemBytes = PL_SMEM;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int i = 3; i >= 0; --i) {
    attr[0].val.clusterDim.x = G << i;
    cfg.gridDim = dim3((G << i) * 64);
    int n = 0;
    KFAC_CUDA(cudaOccupancyMaxActiveClusters(&n, plane_kernel<N, Epi, G>, &cfg));
    room[i] = n > 0 ? n : -1;
  }
  KFAC_REQUIRE(room[0] > 0, "%s: no room for a block", name);
  return KFAC_OK;
}

template <int N, typename Epi>
int plane_launch(const char* name, PlaneLaunch<N>& l, const Epi& epi, bool early,
                 cudaStream_t stream) {
  if (l.n == 0) return KFAC_OK;
  static std::mutex mu;
  static int rooms[64][2][4];                  // by G; 0: not asked yet
  int dev = 0;
  KFAC_CUDA(cudaGetDevice(&dev));
  KFAC_REQUIRE(dev >= 0 && dev < 64, "device index %d unsupported", dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (rooms[dev][1][0] == 0) {
      int room[2][4];
      int rc = plane_prepare<N, Epi, 1>(name, room[0]);
      if (rc == KFAC_OK) rc = plane_prepare<N, Epi, 2>(name, room[1]);
      if (rc != KFAC_OK) return rc;
      for (int k = 0; k < 8; ++k) rooms[dev][k / 4][k % 4] = room[k / 4][k % 4];
    }
  }
  PlaneShape best = {0, 1, 0};
  for (int G = 2; G >= 1; --G) {
    // (where the device counts the rows, as if there were all; a cluster that shares a
    // tile has one, so there a tile has its block or pair)
    plane_number_tiles(l, G);
    const int alone[4] = {rooms[dev][G - 1][0], 0, 0, 0};
    plane_split(l, G, l.rows != nullptr ? alone : rooms[dev][G - 1], best);
  }
  plane_number_tiles(l, best.G);
  l.split = best.split;
  for (int i = 0; i < l.n; ++i) {
    PlaneFields& g = l.p[i].f;
    const int all = (g.K + PL_BK - 1) / PL_BK, each = (all + l.split - 1) / l.split;
    g.odd = best.G == 1 && each <= PL_SHORT ? 0 : 1;
    g.gain = plane_gain(all, each, g.odd + 1);
  }
  const int cluster = best.G * l.split;
  const int clusters =
      l.split > 1 ? l.tiles : std::min(l.tiles, rooms[dev][best.G - 1][0]);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster * clusters);
  cfg.blockDim = dim3(PL_THREADS);
  cfg.dynamicSmemBytes = PL_SMEM;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  if (best.G == 2)
    KFAC_CUDA(cudaLaunchKernelEx(&cfg, plane_kernel<N, Epi, 2>, l, epi));
  else
    KFAC_CUDA(cudaLaunchKernelEx(&cfg, plane_kernel<N, Epi, 1>, l, epi));
  KFAC_LAUNCH_CHECK(name);
  return KFAC_OK;
}

}  // namespace kfac
