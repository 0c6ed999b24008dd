// Orthogonalised updates by Newton-Schulz products: X = G / (|G|_F + eps), then per
// step with X of r rows or columns, whichever are fewer,
//
//   A = X X^T (or X^T X)     B = a I + b A + c A A     X = B X (or X B)
//
// which takes every singular value t of X to a t + b t^3 + c t^5 and leaves the
// singular vectors.  A and B are symmetric: tiles on and below their diagonals, each
// stored with its transpose.
//
// Operands are planes of two fp16 terms (planes.cuh): X 2^13, A 2^12 and B 2^12.  Those
// of 16-bit matrices too: an error of A or B is relative to a I, of order one, and that
// of a single term, 2^-12, is as large as the result's own rounding to fp16 (512 x 4608:
// 8.4e-4 where the rounding makes 2.1e-4); of bf16, and with a second term near B's
// diagonal, it still came to 1.76e-3 where the rounding makes 1.66e-3 (8191 x 2047), and
// to 2.1e-3 for narrow matrices (33 x 385).  So a 16-bit matrix gives what its values
// give in fp32, rounded once.  (With one term where errors are damped 8191 x 2047 took
// 965 us, with two 1713, 4096 x 4096 1850 and 3600.)
//
// Entries of 8 and more in X (16 in A and B) are out of range and give NaN; the
// usual coefficients keep X below 1.3.
//
// Bound: the MMAs.  A step takes r^2 c + r^3 + 2 r^2 c flops, each thrice.
#include <cuda_bf16.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "ortho.cuh"
#include "planes.cuh"

namespace kfac {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormBlocksMax = 512;      // partial sums of a matrix
constexpr long long kNormChunk = 8192;   // elements of a partial sum, at least
// Matrices of one row of launches, whose tables travel as kernel arguments (nothing
// to copy, nothing to keep for a captured graph): up to 4 KB, or up to 32 KB.
constexpr int kFew = 4, kMany = 40;

struct NormJob {
  const void* x;
  Planes out;
  long long count;         // elements
  int rows, cols;
  int norm_begin, norm_blocks;
  int pack_begin;          // first block of the pack launch
};

template <int N>
struct NormLaunch {
  NormJob j[N];
  int n;
  double eps;
  double* part;
};

template <typename T> __device__ __forceinline__ float as_float(T x);
template <> __device__ __forceinline__ float as_float(float x) { return x; }
template <> __device__ __forceinline__ float as_float(__half x) {
  return __half2float(x);
}
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) {
  return __float2half_rn(x);
}
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) {
  return __float2bfloat16_rn(x);
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kNormThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kNormThreads / 32; ++w) v += part[w];
  return v;
}

// Eight values from x[0..], zeros past `live`.
template <typename T>
__device__ __forceinline__ void load8(const T* x, int live, bool vec, float (&v)[8]) {
  if (vec && live >= 8) {
    constexpr int W = 16 / sizeof(T);        // values of a 16-byte word
    struct alignas(16) Word { T x[W]; };
#pragma unroll
    for (int k = 0; k < 8 / W; ++k) {
      const Word w = reinterpret_cast<const Word*>(x)[k];
#pragma unroll
      for (int e = 0; e < W; ++e) v[W * k + e] = as_float(w.x[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < live ? as_float(x[e]) : 0.f;
  }
}

// Sums of squares, in fp64: no size of the elements is out of range.
template <int N, typename T>
__global__ void __launch_bounds__(kNormThreads)
ortho_norm_kernel(const __grid_constant__ NormLaunch<N> l) {
  int f = 0;
  for (int i = 1; i < l.n; ++i)
    if (l.j[i].norm_begin <= (int)blockIdx.x) f = i;
  const NormJob& j = l.j[f];
  const T* x = static_cast<const T*>(j.x);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const long long words = (j.count + 7) >> 3;
  double sum = 0;
  for (long long w = (long long)(blockIdx.x - j.norm_begin) * kNormThreads + threadIdx.x;
       w < words; w += (long long)j.norm_blocks * kNormThreads) {
    float v[8];
    load8(x + 8 * w, (int)min(8LL, j.count - 8 * w), vec, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fma((double)v[e], (double)v[e], sum);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) l.part[blockIdx.x] = sum;
}

constexpr int kPackWords = 4;            // words of eight values a thread

// X = G / (|G| + eps), as planes.
template <int N, typename T>
__global__ void __launch_bounds__(kNormThreads)
ortho_pack_kernel(const __grid_constant__ NormLaunch<N> l) {
  let_next_launch_begin();
  wait_for_launch_before();
  int f = 0;
  for (int i = 1; i < l.n; ++i)
    if (l.j[i].pack_begin <= (int)blockIdx.x) f = i;
  const NormJob& j = l.j[f];
  double sum = 0;
  for (int b = threadIdx.x; b < j.norm_blocks; b += kNormThreads)
    sum += l.part[j.norm_begin + b];
  const double s = (double)(1 << kXExp) / (sqrt(block_sum(sum)) + l.eps);
  const int words = j.out.ld >> 3;       // of a row
  const T* x = static_cast<const T*>(j.x);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                   (j.cols * (int)sizeof(T)) % 16 == 0;
  const long long total = (long long)j.rows * words;
  const long long w0 =
      (long long)(blockIdx.x - j.pack_begin) * kNormThreads * kPackWords + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kPackWords; ++u) {
    const long long w = w0 + u * kNormThreads;
    if (w >= total) break;
    const long long r = w / words;
    const int c = 8 * (int)(w - r * words);
    float v[8];
    load8(x + r * j.cols + c, j.cols - c, vec, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(v[e] * s);
    uint4 hi, lo;
    pl_split2(v[0], v[1], hi.x, lo.x);
    pl_split2(v[2], v[3], hi.y, lo.y);
    pl_split2(v[4], v[5], hi.z, lo.z);
    pl_split2(v[6], v[7], hi.w, lo.w);
    __half* to = j.out.p + r * j.out.ld + c;
    *reinterpret_cast<uint4*>(to) = hi;
    *reinterpret_cast<uint4*>(to + j.out.plane) = lo;
  }
}

// alpha * sums, with `poly` plus beta * `add` and `diag` on the diagonal, as planes.
struct EpiPlanes {
  float alpha, beta, diag;
  bool poly;
  __device__ __forceinline__ NothingAhead begin(const PlaneFields&,
                                                const PlaneTile&) const {
    return NothingAhead();
  }
  __device__ __forceinline__ void store(const PlaneFields& g, const PlaneTile& t,
                                        float (&v)[32], bool mirror,
                                        NothingAhead) const {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= alpha * g.gain;
    if (poly) {
      // `add` in the registers' order, by way of shared memory
      const int j = t.lane & 3, r = t.lane >> 2;
      const unsigned piece = smem_u32(t.piece);
      const __half* p = g.add.p + (long long)(t.r0 + r) * g.add.ld + t.c0 + 8 * j;
      const bool in = t.c0 + 8 * j < g.N;
      uint4 w[2][4];
#pragma unroll
      for (int term = 0; term < 2; ++term)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[term][i] = make_uint4(0, 0, 0, 0);
          if (in && t.r0 + r + 8 * i < g.M)
            w[term][i] = *reinterpret_cast<const uint4*>(
                p + (term ? g.add.plane : 0) + 8LL * i * g.add.ld);
        }
      __syncwarp();
#pragma unroll
      for (int term = 0; term < 2; ++term)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                       ::"r"(piece + 2048 * term + 512 * i + row64_off(r, j)),
                         "r"(w[term][i].x), "r"(w[term][i].y), "r"(w[term][i].z),
                         "r"(w[term][i].w)
                       : "memory");
      __syncwarp();
#pragma unroll
      for (int term = 0; term < 2; ++term)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          unsigned x[4];                 // rows' eighths
          ld_matrix(piece + 2048 * term + row64_off(t.lane, k), x[0], x[1], x[2], x[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x[e]));
            const int at = 16 * (e >> 1) + 4 * k + 2 * (e & 1);
            v[at] = fmaf(beta, y.x, v[at]);
            v[at + 1] = fmaf(beta, y.y, v[at + 1]);
          }
        }
      // (rows and columns past the matrix: of no matter)
      if (t.r0 == t.c0) {
        const int d = 2 * (t.lane & 3) - (t.lane >> 2);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (16 * (i >> 4) + 8 * ((i >> 1) & 1) - 8 * ((i >> 2) & 3) - (i & 1) == d)
            v[i] += diag;
      }
    }
    pl_store_planes(t, g.out, v, g.M, g.N, mirror);
  }
};

// The last step: out = scale * X, and W = keep * W - lr * scale * X.
template <typename T>
struct EpiLast {
  float alpha, keep, lr;
  __device__ __forceinline__ NothingAhead begin(const PlaneFields&,
                                                const PlaneTile&) const {
    return NothingAhead();
  }
  __device__ __forceinline__ void store(const PlaneFields& g, const PlaneTile& t,
                                        float (&v)[32], bool, NothingAhead) const {
    const unsigned piece = smem_u32(t.piece);
    T* const dst = static_cast<T*>(g.dst);
    T* const param = static_cast<T*>(g.param);
    const float a = alpha * g.gain * g.scale;
    const int lane = t.lane, N = g.N, rows = g.M - t.r0;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= a;
    __syncwarp();
    pl_put_floats(piece, v, lane);
    __syncwarp();
    constexpr int W = 16 / sizeof(T);      // values of a 16-byte word
    const bool words =
        N % W == 0 && ((reinterpret_cast<uintptr_t>(dst) |
                        reinterpret_cast<uintptr_t>(param)) & 15) == 0;
    if (words) {
      struct alignas(16) Word { T x[W]; };
      constexpr int L = 32 / W, R = 32 / L;          // lanes of a row, rows at a time
      const int c = t.c0 + W * (lane % L), r = lane / L;
      if (c >= N) return;
      const long long first = (long long)(t.r0 + r) * N + c, step = (long long)R * N;
#pragma unroll
      for (int i = 0; i < 32 / R; ++i) {
        if (r + R * i >= rows) break;
        alignas(16) float x[W];
#pragma unroll
        for (int k = 0; k < W / 4; ++k)
          *reinterpret_cast<float4*>(&x[4 * k]) =
              pl_word(piece, r + R * i, W / 4 * (lane % L) + k);
        Word o;
        if (dst != nullptr) {
#pragma unroll
          for (int e = 0; e < W; ++e) o.x[e] = from_float<T>(x[e]);
          *reinterpret_cast<Word*>(dst + first + step * i) = o;
        }
        if (param != nullptr) {
          o = *reinterpret_cast<const Word*>(param + first + step * i);
#pragma unroll
          for (int e = 0; e < W; ++e)
            o.x[e] = from_float<T>(fmaf(keep, as_float(o.x[e]), -lr * x[e]));
          *reinterpret_cast<Word*>(param + first + step * i) = o;
        }
      }
      return;
    }
    const int c = t.c0 + lane;
    if (c >= N) return;
    const long long first = (long long)t.r0 * N + c;
#pragma unroll 4
    for (int i = 0; i < min(rows, 32); ++i) {
      const float x = pl_float(piece, i, lane);
      const long long k = first + (long long)i * N;
      if (dst != nullptr) dst[k] = from_float<T>(x);
      if (param != nullptr)
        param[k] = from_float<T>(fmaf(keep, as_float(param[k]), -lr * x));
    }
  }
};

// ----------------------------------------------------------------- host side

struct Shape {
  int rows, cols, small;      // small: the shorter side
  Planes x[2], a, b;
};

int up8(int v) { return (v + 7) & ~7; }
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

Planes place(char* ws, size_t& at, int rows, int cols) {
  Planes p;
  p.ld = up8(cols);
  p.plane = (long long)rows * p.ld;
  p.p = reinterpret_cast<__half*>(ws + at);
  at += up256((size_t)p.plane * 4);
  return p;
}

int norm_blocks_of(long long count) {
  return (int)std::max<long long>(
      1, std::min<long long>(kNormBlocksMax, (count + kNormChunk - 1) / kNormChunk));
}

// Whether every matrix is one that a block or a cluster orthogonalises by itself.
// Beside larger ones they ride along in the products' launches, which take no longer
// for them.
bool all_small(int count, const int* rows, const int* cols) {
  for (int i = 0; i < count; ++i)
    if (std::min(rows[i], cols[i]) > kSmallShort ||
        std::max(rows[i], cols[i]) > kSmallClusterLong)
      return false;
  return true;
}

// Lays the matrices' planes out behind `ws`; the bytes they take.
size_t lay_out(int count, const int* rows, const int* cols, char* ws,
               std::vector<Shape>* shapes) {
  if (all_small(count, rows, cols)) return 0;
  size_t at = 0;
  long long parts = 0;
  for (int i = 0; i < count; ++i)
    parts += norm_blocks_of((long long)rows[i] * cols[i]);
  at += up256((size_t)parts * sizeof(double));
  for (int i = 0; i < count; ++i) {
    Shape s;
    s.rows = rows[i];
    s.cols = cols[i];
    s.small = std::min(rows[i], cols[i]);
    for (int k = 0; k < 2; ++k) s.x[k] = place(ws, at, s.rows, s.cols);
    s.a = place(ws, at, s.small, s.small);
    s.b = place(ws, at, s.small, s.small);
    if (shapes != nullptr) shapes->push_back(s);
  }
  return at + 256;            // (the workspace may begin anywhere)
}

struct Call {
  int dtype, steps;
  const float* coefficients;
  float eps, lr, decay;
  const void* const* x;
  void* const* out;
  void* const* param;
  const float* scale;
};

template <int N, typename T>
int launch_last(PlaneLaunch<N>& l, const Call& c, cudaStream_t st) {
  const EpiLast<T> epi = {exp2f(-(kXExp + kAExp)), 1.f - c.lr * c.decay, c.lr};
  return plane_launch("ortho last product", l, epi, true, st);
}

template <int N, typename T>
int launch_norm(const NormLaunch<N>& l, int norm_blocks, int pack_blocks,
                cudaStream_t st) {
  ortho_norm_kernel<N, T><<<norm_blocks, kNormThreads, 0, st>>>(l);
  KFAC_LAUNCH_CHECK("ortho_norm_kernel");
  return launch_behind("ortho_pack_kernel", true, ortho_pack_kernel<N, T>, pack_blocks,
                       kNormThreads, 0, st, l);
}

int run_small(int count, const int* rows, const int* cols, const Call& c,
              void* stream) {
  SmallLaunch l;
  l.steps = c.steps;
  l.eps = c.eps;
  l.keep = 1.f - c.lr * c.decay;
  l.lr = c.lr;
  std::copy(c.coefficients, c.coefficients + 3 * c.steps, l.coefficients);
  for (int first = 0; first < count; first += kSmallJobs) {
    l.n = std::min(kSmallJobs, count - first);
    for (int k = 0; k < l.n; ++k) {
      const int i = first + k;
      l.j[k] = {c.x[i], c.out != nullptr ? c.out[i] : nullptr,
                c.param != nullptr ? c.param[i] : nullptr, rows[i], cols[i],
                c.scale[i]};
    }
    const int rc = launch_ortho_small(l, c.dtype, (cudaStream_t)stream);
    if (rc != KFAC_OK) return rc;
  }
  return KFAC_OK;
}

// All launches of up to N matrices, numbers first .. first + n of the call.
template <int N>
int run_group(const Shape* s, int first, int n, double* part, const Call& c,
              cudaStream_t st) {
  NormLaunch<N> nl;
  nl.n = n;
  nl.eps = c.eps;
  nl.part = part;
  long long norm_blocks = 0, pack_blocks = 0;
  for (int i = 0; i < n; ++i) {
    NormJob& j = nl.j[i];
    j.x = c.x[first + i];
    j.out = s[i].x[0];
    j.rows = s[i].rows;
    j.cols = s[i].cols;
    j.count = (long long)j.rows * j.cols;
    j.norm_begin = (int)norm_blocks;
    j.norm_blocks = norm_blocks_of(j.count);
    norm_blocks += j.norm_blocks;
    j.pack_begin = (int)pack_blocks;
    pack_blocks += ((long long)j.rows * (j.out.ld / 8) + kNormThreads * kPackWords - 1) /
                   (kNormThreads * kPackWords);
    KFAC_REQUIRE(pack_blocks < (1LL << 31), "orthogonalize: too many elements");
  }
  int rc = c.dtype == KFAC_WIRE_F32
               ? launch_norm<N, float>(nl, (int)norm_blocks, (int)pack_blocks, st)
           : c.dtype == KFAC_WIRE_F16
               ? launch_norm<N, __half>(nl, (int)norm_blocks, (int)pack_blocks, st)
               : launch_norm<N, __nv_bfloat16>(nl, (int)norm_blocks, (int)pack_blocks,
                                               st);
  if (rc != KFAC_OK) return rc;

  // the three products of a step, with X in either of its places
  PlaneLaunch<N> gram[2], poly, apply[2];
  for (int i = 0; i < n; ++i) {
    const Shape& m = s[i];
    const bool tall = m.rows > m.cols;
    const int r = m.small;
    PlaneFields g = {};
    g.scale = c.scale[first + i];
    g.dst = c.out != nullptr ? c.out[first + i] : nullptr;
    g.param = c.param != nullptr ? c.param[first + i] : nullptr;
    CUtensorMap along[2], down[2], a, b;
    for (int k = 0; k < 2; ++k) {
      if ((rc = plane_map(&along[k], m.x[k], m.rows, m.cols, false)) != KFAC_OK ||
          (rc = plane_map(&down[k], m.x[k], m.rows, m.cols, true)) != KFAC_OK)
        return rc;
    }
    if ((rc = plane_map(&a, m.a, r, r, false)) != KFAC_OK ||
        (rc = plane_map(&b, m.b, r, r, false)) != KFAC_OK)
      return rc;
    for (int k = 0; k < 2; ++k) {
      gram[k].p[i].ma = gram[k].p[i].mb = tall ? down[k] : along[k];
      PlaneFields& p = gram[k].p[i].f;
      p = g;
      p.a_mn = p.b_mn = tall;
      p.M = p.N = r;
      p.K = tall ? m.rows : m.cols;
      p.lower = p.same = 1;
      p.out = m.a;
      apply[k].p[i].ma = tall ? along[k] : b;
      apply[k].p[i].mb = tall ? b : down[k];
      PlaneFields& q = apply[k].p[i].f;
      q = g;
      q.M = m.rows;
      q.N = m.cols;
      q.K = r;
      q.b_mn = !tall;
      q.out = m.x[k ^ 1];
    }
    poly.p[i].ma = poly.p[i].mb = a;
    PlaneFields& p = poly.p[i].f;
    p = g;
    p.M = p.N = p.K = r;
    p.lower = p.same = 1;
    p.out = m.b;
    p.add = m.a;
  }
  for (int k = 0; k < 2; ++k) {
    gram[k].n = apply[k].n = n;
    gram[k].rows = apply[k].rows = nullptr;
  }
  poly.n = n;
  poly.rows = nullptr;
  for (int step = 0; step < c.steps; ++step) {
    const float* k = c.coefficients + 3 * step;
    const int from = step & 1;
    const EpiPlanes make_a = {exp2f(kAExp - 2 * kXExp), 0.f, 0.f, false};
    rc = plane_launch("ortho X X^T", gram[from], make_a, true, st);
    if (rc != KFAC_OK) return rc;
    const EpiPlanes make_b = {k[2] * exp2f(-kAExp), k[1], k[0] * exp2f(kAExp), true};
    rc = plane_launch("ortho A A", poly, make_b, true, st);
    if (rc != KFAC_OK) return rc;
    if (step + 1 < c.steps) {
      const EpiPlanes make_x = {exp2f(-kAExp), 0.f, 0.f, false};
      rc = plane_launch("ortho B X", apply[from], make_x, true, st);
    } else if (c.dtype == KFAC_WIRE_F32) {
      rc = launch_last<N, float>(apply[from], c, st);
    } else if (c.dtype == KFAC_WIRE_F16) {
      rc = launch_last<N, __half>(apply[from], c, st);
    } else {
      rc = launch_last<N, __nv_bfloat16>(apply[from], c, st);
    }
    if (rc != KFAC_OK) return rc;
  }
  return KFAC_OK;
}

}  // namespace
}  // namespace kfac

using namespace kfac;

namespace kfac {
int ortho_status_read(int* out) {
  KFAC_CUDA(cudaMemcpyFromSymbol(out, g_plane_status, sizeof(int)));
  return KFAC_OK;
}
}  // namespace kfac

static int check_shapes(int count, const int* rows, const int* cols) {
  KFAC_REQUIRE(count >= 0, "orthogonalize: %d matrices", count);
  KFAC_REQUIRE(count == 0 || (rows != nullptr && cols != nullptr),
               "orthogonalize: null pointer");
  for (int i = 0; i < count; ++i) {
    KFAC_REQUIRE(rows[i] >= 1 && cols[i] >= 1 && rows[i] <= (1 << 20) &&
                     cols[i] <= (1 << 20),
                 "orthogonalize: matrix %d is %d x %d (1 .. 2^20 a side)", i, rows[i],
                 cols[i]);
  }
  return KFAC_OK;
}

// What a call writes may be what it reads of the same matrix, and nothing else: a
// matrix may still be read, or be written by others, while one is written.
static int check_apart(int count, const int* rows, const int* cols, size_t size,
                       const Call& c) {
  struct Piece {
    uintptr_t begin, end;
    int matrix;
    bool written;
  };
  std::vector<Piece> all;
  all.reserve(3 * (size_t)count);
  auto add = [&](const void* p, int i, bool written) -> int {
    if (p == nullptr) return KFAC_OK;
    KFAC_REQUIRE(aligned_to(p, size), "orthogonalize: matrix %d is not aligned", i);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    all.push_back({at, at + (size_t)rows[i] * cols[i] * size, i, written});
    return KFAC_OK;
  };
  for (int i = 0; i < count; ++i) {
    int rc = add(c.x[i], i, false);
    if (rc == KFAC_OK && c.out != nullptr) rc = add(c.out[i], i, true);
    if (rc == KFAC_OK && c.param != nullptr) rc = add(c.param[i], i, true);
    if (rc != KFAC_OK) return rc;
  }
  std::sort(all.begin(), all.end(),
            [](const Piece& a, const Piece& b) { return a.begin < b.begin; });
  for (size_t i = 0; i < all.size(); ++i)
    for (size_t k = i + 1; k < all.size() && all[k].begin < all[i].end; ++k) {
      const Piece &a = all[i], &b = all[k];
      KFAC_REQUIRE((!a.written && !b.written) ||
                       (a.written != b.written && a.matrix == b.matrix &&
                        a.begin == b.begin),
                   "orthogonalize: what is written of matrix %d overlaps matrix %d",
                   a.written ? a.matrix : b.matrix, a.written ? b.matrix : a.matrix);
    }
  return KFAC_OK;
}

extern "C" size_t kfac_orthogonalize_workspace_bytes(int count, const int* rows,
                                                     const int* cols) {
  if (count <= 0 || check_shapes(count, rows, cols) != KFAC_OK) return 0;
  return lay_out(count, rows, cols, nullptr, nullptr);
}

extern "C" int kfac_orthogonalize(int dtype, int count, const int* rows,
                                  const int* cols, const void* const* x,
                                  void* const* out, void* const* param,
                                  const float* scale, int steps,
                                  const float* coefficients, float eps, float lr,
                                  float decay, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc = check_shapes(count, rows, cols);
  if (rc != KFAC_OK) return rc;
  KFAC_REQUIRE(dtype == KFAC_WIRE_F32 || dtype == KFAC_WIRE_F16 ||
                   dtype == KFAC_WIRE_BF16,
               "orthogonalize: unknown element type %d", dtype);
  KFAC_REQUIRE(steps >= 1 && steps <= kStepsMax, "orthogonalize: %d steps (1 .. %d)",
               steps, kStepsMax);
  KFAC_REQUIRE(eps >= 0.f, "orthogonalize: eps is %g", (double)eps);
  if (count == 0) return KFAC_OK;
  KFAC_REQUIRE(x != nullptr && scale != nullptr && coefficients != nullptr &&
                   (out != nullptr || param != nullptr),
               "orthogonalize: null pointer");
  for (int i = 0; i < count; ++i)
    KFAC_REQUIRE(x[i] != nullptr && ((out != nullptr && out[i] != nullptr) ||
                                     (param != nullptr && param[i] != nullptr)),
                 "orthogonalize: matrix %d is null, or has nowhere to go", i);
  try {
    const Call c = {dtype, steps, coefficients, eps, lr, decay, x, out, param, scale};
    const size_t need = lay_out(count, rows, cols, nullptr, nullptr);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
      return fail(KFAC_ERR_WORKSPACE,
                  "orthogonalize: %zu bytes of workspace, %zu needed",
                  workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    rc = check_apart(count, rows, cols, dtype == KFAC_WIRE_F32 ? 4 : 2, c);
    if (rc != KFAC_OK) return rc;
    if (need == 0) return run_small(count, rows, cols, c, stream);
    char* ws = reinterpret_cast<char*>(
        (reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
    std::vector<Shape> shapes;
    shapes.reserve(count);
    lay_out(count, rows, cols, ws, &shapes);
    double* part = reinterpret_cast<double*>(ws);
    cudaStream_t st = (cudaStream_t)stream;
    for (int i = 0; i < count;) {
      const int left = count - i;
      const int n = left <= kFew ? left : std::min(left, kMany);
      rc = n <= kFew ? run_group<kFew>(&shapes[i], i, n, part, c, st)
                     : run_group<kMany>(&shapes[i], i, n, part, c, st);
      if (rc != KFAC_OK) return rc;
      for (int k = 0; k < n; ++k)
        part += norm_blocks_of((long long)rows[i + k] * cols[i + k]);
      i += n;
    }
  } catch (const std::exception& e) {
    return fail(KFAC_ERR_INVALID, "orthogonalize: %s", e.what());
  }
  return KFAC_OK;
}
