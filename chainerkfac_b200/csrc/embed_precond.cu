// The K-FAC step of a token embedding (vocab x width), a fully connected layer on rows
// with a single one: its input factor is a diagonal, so
//
//   kf = diag(1 / (A + delta)) grad G_inv,  v = momentum v - lr kf,  W = W + v.
//
// A batch reaches few of the tokens.  The first launch reads the gradient once, a row a
// warp: a row of zeros has its update at once (kf = 0), any other goes as two fp16
// terms, scaled by its own power of two, into the next free row of the planes
// (planes.cuh) that are multiplied by G_inv; which row of the planes makes no
// difference to its values.  The second launch multiplies as many rows as there are,
// and its epilogue scales and scatters them; the third updates their weights.  (In that
// epilogue an SM has to store three rows where it now stores one, 32 bytes a cycle:
// 32000 x 1024 with 12 800 rows took 209 us so and 192 apart; 8000 x 256 with 300 rows,
// four SMs at work, 36 and 29.)
//
// Bound: HBM, 24 bytes an element (gradient in, kf out, velocity and weight in and
// out), where the batch reaches few tokens; else the products, three MMAs each.
#include <algorithm>

#include "planes.cuh"

namespace kfac {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTopExp = 14;        // a row's largest value: 2^14 and more, below 2^15

struct EmbedStep {
  const float* G;                  // width x width, symmetric
  const float* A;
  const float* damping;            // one value
  const float* grad;
  float* kf;
  float* param;                    // or null, with mom
  float* mom;
  float lr, momentum;
  int vocab, width;
  Planes rows, g;
  int* count;                      // rows of `rows`
  int* index;                      // their tokens
  int* row_exp;                    // of a row of `rows`
  int* col_exp;                    // of a row (and column) of G
  bool vec;                        // all rows begin at 16 bytes
  bool even;                       // kf, weights and velocities lie alike within 16 bytes
};

// A row of floats as up to three in front, words of 16 bytes, and up to three behind.
struct RowWords {
  int head, words, tail;
};
__device__ __forceinline__ RowWords row_words(const float* x, int width) {
  RowWords w;
  w.head = min((int)((-reinterpret_cast<uintptr_t>(x) & 15) >> 2), width);
  w.words = (width - w.head) >> 2;
  w.tail = width - w.head - 4 * w.words;
  return w;
}

// Exponent of a row's largest value, by a warp; kNoExp: zeros.
__device__ __forceinline__ int row_top(const float* x, int width, int lane) {
  const RowWords w = row_words(x, width);
  int top = kNoExp;
  if (lane < w.head) top = exp_of(x[lane]);
  if (lane < w.tail) top = max(top, exp_of(x[w.head + 4 * w.words + lane]));
  const float4* const x4 = reinterpret_cast<const float4*>(x + w.head);
#pragma unroll 1
  for (int k0 = lane; k0 < w.words; k0 += 256) {
    float4 y[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) y[u] = x4[min(k0 + 32 * u, w.words - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      top = max(top, max(max(exp_of(y[u].x), exp_of(y[u].y)),
                         max(exp_of(y[u].z), exp_of(y[u].w))));
  }
  return __reduce_max_sync(0xffffffffu, top);
}

// x 2^s as planes, row `to`.
__device__ __forceinline__ void pack_planes(const float* x, int width, bool vec,
                                            const Planes& o, int to, int s, int lane) {
  __half* const hi = o.p + (long long)to * o.ld;
#pragma unroll 4
  for (int k = 4 * lane; k < width; k += 128) {
    float y[4];
    if (vec) {
      const float4 w = *reinterpret_cast<const float4*>(x + k);
      y[0] = w.x; y[1] = w.y; y[2] = w.z; y[3] = w.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = k + e < width ? x[k + e] : 0.f;
    }
    uint2 h, l;
    pl_split2(scale_exp(y[0], s), scale_exp(y[1], s), h.x, l.x);
    pl_split2(scale_exp(y[2], s), scale_exp(y[3], s), h.y, l.y);
    *reinterpret_cast<uint2*>(hi + k) = h;
    *reinterpret_cast<uint2*>(hi + o.plane + k) = l;
  }
}

// The update of a row: with its kf (GRADIENT), or without a gradient, kf = 0.
template <bool GRADIENT>
__device__ __forceinline__ void update_row(const EmbedStep& e, long long at, int lane) {
  float* const kf = e.kf + at;
  float* const mom = e.param != nullptr ? e.mom + at : nullptr;
  float* const param = e.param != nullptr ? e.param + at : nullptr;
  auto one = [&](int k) {
    if (!GRADIENT) kf[k] = 0.f;
    if (param == nullptr) return;
    const float v = e.momentum * mom[k] - (GRADIENT ? e.lr * kf[k] : 0.f);
    mom[k] = v;
    param[k] += v;
  };
  if (!e.even) {
#pragma unroll 4
    for (int k = lane; k < e.width; k += 32) one(k);
    return;
  }
  const RowWords w = row_words(kf, e.width);
  if (lane < w.head) one(lane);
  if (lane < w.tail) one(w.head + 4 * w.words + lane);
  float4* const kf4 = reinterpret_cast<float4*>(kf + w.head);
  float4* const mom4 = reinterpret_cast<float4*>(mom + w.head);
  float4* const param4 = reinterpret_cast<float4*>(param + w.head);
#pragma unroll 1
  for (int k0 = lane; k0 < w.words; k0 += 128) {
    float4 x[4], v[4], p[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = min(k0 + 32 * u, w.words - 1);
      if (GRADIENT) x[u] = kf4[k];
      if (param == nullptr) continue;
      v[u] = mom4[k];
      p[u] = param4[k];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + 32 * u;
      if (k >= w.words) break;
      if (!GRADIENT) kf4[k] = x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (param == nullptr) continue;
      v[u].x = e.momentum * v[u].x - e.lr * x[u].x;
      v[u].y = e.momentum * v[u].y - e.lr * x[u].y;
      v[u].z = e.momentum * v[u].z - e.lr * x[u].z;
      v[u].w = e.momentum * v[u].w - e.lr * x[u].w;
      mom4[k] = v[u];
      p[u].x += v[u].x;
      p[u].y += v[u].y;
      p[u].z += v[u].z;
      p[u].w += v[u].w;
      param4[k] = p[u];
    }
  }
}

__global__ void __launch_bounds__(kThreads)
embed_rows_kernel(const __grid_constant__ EmbedStep e) {
  let_next_launch_begin();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * kWarps;
  // the rows of G first, then the gradient's
  for (long long i = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
       i < (long long)e.width + e.vocab; i += step) {
    const bool of_g = i < e.width;
    const long long row = of_g ? i : i - e.width;
    const float* x = (of_g ? e.G : e.grad) + row * e.width;
    const int top = row_top(x, e.width, lane);
    if (top == kNoExp && !of_g) {
      update_row<false>(e, row * e.width, lane);
      continue;
    }
    const int s = top == kNoExp ? 0 : kTopExp - top;
    int to = (int)row;
    if (!of_g) {
      if (lane == 0) to = atomicAdd(e.count, 1);
      to = __shfl_sync(0xffffffffu, to, 0);
    }
    pack_planes(x, e.width, e.vec, of_g ? e.g : e.rows, to, s, lane);
    if (lane == 0) {
      (of_g ? e.col_exp : e.row_exp)[to] = -s;
      if (!of_g) e.index[to] = (int)row;
    }
  }
}

struct EpiEmbed {
  EmbedStep e;

  // Of row `lane`: its token, exponent and divisor.
  struct Row {
    int token, exp;
    float inv;
  };
  __device__ __forceinline__ Row begin(const PlaneFields& g, const PlaneTile& t) const {
    Row o;
    const int r = max(min(t.r0 + t.lane, g.M - 1), 0);
    o.token = e.index[r];
    o.exp = e.row_exp[r];
    o.inv = 1.f / (e.A[o.token] + *e.damping);
    return o;
  }

  __device__ __forceinline__ void store(const PlaneFields& g, const PlaneTile& t,
                                        float (&v)[32], bool, const Row& ahead) const {
    const unsigned piece = smem_u32(t.piece);
    const int lane = t.lane, width = e.width;
    const int token = ahead.token, re = ahead.exp;
    const float inv = ahead.inv;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= g.gain;
    __syncwarp();
    pl_put_floats(piece, v, lane);
    __syncwarp();
    const int rows = min(32, g.M - t.r0);
    // Two factors, of the column and of the row, where neither they nor their product
    // (2^-120 .. 2^120) can leave the range; else exponents added up for a value.  Which
    // of them depends on its own row and column only, not on the rows beside it.
    const int c1 = t.c0 + lane, ce1 = c1 < width ? e.col_exp[c1] : 0;
    const float row_f = scale_exp(inv, re), col_f = scale_exp(1.f, ce1);
    const bool near_row = abs(re) <= 60 && row_f >= 1e-18f && row_f <= 1e18f;
    const bool near_col = abs(ce1) <= 60;
    const unsigned near_rows = __ballot_sync(0xffffffffu, near_row);
    if (e.vec && near_rows == 0xffffffffu && __all_sync(0xffffffffu, near_col)) {
      const int c = t.c0 + 4 * (lane & 7);
      float4 f4;
      f4.x = __shfl_sync(0xffffffffu, col_f, 4 * (lane & 7));
      f4.y = __shfl_sync(0xffffffffu, col_f, 4 * (lane & 7) + 1);
      f4.z = __shfl_sync(0xffffffffu, col_f, 4 * (lane & 7) + 2);
      f4.w = __shfl_sync(0xffffffffu, col_f, 4 * (lane & 7) + 3);
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const int row = i + (lane >> 3);
        const float f = __shfl_sync(0xffffffffu, row_f, row);
        const int to = __shfl_sync(0xffffffffu, token, row);
        float4 x = pl_word(piece, row, lane & 7);
        x.x *= f4.x * f;
        x.y *= f4.y * f;
        x.z *= f4.z * f;
        x.w *= f4.w * f;
        if (c < width && row < rows)
          *reinterpret_cast<float4*>(e.kf + (long long)to * width + c) = x;
      }
      return;
    }
#pragma unroll 8
    for (int row = 0; row < rows; ++row) {
      const int to = __shfl_sync(0xffffffffu, token, row);
      const int n = __shfl_sync(0xffffffffu, re, row);
      const float f = __shfl_sync(0xffffffffu, row_f, row);
      const float d = __shfl_sync(0xffffffffu, inv, row);
      float x = pl_float(piece, row, lane);
      x = near_col && ((near_rows >> row) & 1) ? x * (col_f * f)
                                               : scale_exp(x, n + ce1) * d;
      if (c1 < width) e.kf[(long long)to * width + c1] = x;
    }
  }
};

// The momentum update of the rows that have a gradient, a row a warp.
__global__ void __launch_bounds__(kThreads)
embed_update_kernel(const __grid_constant__ EmbedStep e) {
  wait_for_launch_before();
  const int rows = *reinterpret_cast<const volatile int*>(e.count);
  for (int r = blockIdx.x * kWarps + (threadIdx.x >> 5); r < rows;
       r += gridDim.x * kWarps)
    update_row<true>(e, (long long)e.index[r] * e.width, threadIdx.x & 31);
}

long long parts_of(long long a, long long b) { return (a + b - 1) / b; }

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

Planes place(char* ws, size_t& at, long long rows, int cols) {
  Planes p;
  p.ld = (cols + 7) & ~7;
  p.plane = rows * p.ld;
  p.p = reinterpret_cast<__half*>(ws + at);
  at += up256((size_t)p.plane * 4);
  return p;
}

// Lays a call's scratch out behind `ws`; the bytes it takes.
size_t lay_out(int64_t vocab, int width, char* ws, EmbedStep* e) {
  size_t at = 0;
  const Planes rows = place(ws, at, vocab, width), g = place(ws, at, width, width);
  int* const ints = reinterpret_cast<int*>(ws + at);
  const size_t v = up256((size_t)vocab * 4), w = up256((size_t)width * 4);
  at += 256 + 2 * v + w;
  if (e != nullptr) {
    e->rows = rows;
    e->g = g;
    e->count = ints;
    e->index = ints + 64;
    e->row_exp = ints + 64 + v / 4;
    e->col_exp = ints + 64 + 2 * (v / 4);
  }
  return at + 256;            // (the workspace may begin anywhere)
}

int check_shape(int64_t vocab, int width) {
  KFAC_REQUIRE(vocab >= 1 && vocab < (1LL << 31) - 256 && width >= 1 &&
                   width <= (1 << 20),
               "precondition_embedding: a weight of %lld x %d", (long long)vocab, width);
  // (tiles are numbered in 32 bits)
  KFAC_REQUIRE(((vocab + 255) / 256) * (int64_t)((width + 255) / 256) < (1LL << 31),
               "precondition_embedding: a weight of %lld x %d", (long long)vocab, width);
  return KFAC_OK;
}

}  // namespace

int embed_status_read(int* out) {
  KFAC_CUDA(cudaMemcpyFromSymbol(out, g_plane_status, sizeof(int)));
  return KFAC_OK;
}

}  // namespace kfac

using namespace kfac;

extern "C" size_t kfac_precondition_embedding_workspace_bytes(int64_t vocab,
                                                              int width) {
  return check_shape(vocab, width) == KFAC_OK ? lay_out(vocab, width, nullptr, nullptr)
                                              : 0;
}

extern "C" int kfac_precondition_embedding(int64_t vocab, int width, const float* G_inv,
                                           const float* A, const float* damping,
                                           const float* grad, float* kf, float* param,
                                           float* mom, float lr, float momentum,
                                           void* workspace, size_t workspace_bytes,
                                           void* stream) {
  int rc = check_shape(vocab, width);
  if (rc != KFAC_OK) return rc;
  KFAC_REQUIRE(G_inv != nullptr && A != nullptr && damping != nullptr &&
                   grad != nullptr && kf != nullptr,
               "precondition_embedding: null pointer");
  KFAC_REQUIRE((param == nullptr) == (mom == nullptr),
               "precondition_embedding: a weight and its velocity go together");
  const size_t need = lay_out(vocab, width, nullptr, nullptr);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(KFAC_ERR_WORKSPACE,
                "precondition_embedding: %zu bytes of workspace, %zu needed",
                workspace == nullptr ? (size_t)0 : workspace_bytes, need);
  // (kf may be where the gradient was: a row is read before its kf is there)
  const size_t all = (size_t)vocab * width * sizeof(float);
  struct Piece {
    const void* p;
    size_t bytes;
    bool written;
  };
  const Piece pieces[] = {{kf, all, true},
                          {param, all, true},
                          {mom, all, true},
                          {grad, all, false},
                          {G_inv, (size_t)width * width * sizeof(float), false},
                          {A, (size_t)vocab * sizeof(float), false},
                          {damping, sizeof(float), false},
                          {workspace, need, false}};
  for (const Piece& a : pieces) {
    KFAC_REQUIRE(a.p == workspace || aligned_to(a.p, sizeof(float)),
                 "precondition_embedding: arrays not aligned to 4 bytes");
    for (const Piece* b = &a + 1; b != pieces + 8; ++b)
      KFAC_REQUIRE(!a.written || (a.p == kf && b->p == grad && kf == grad) ||
                       !overlap(a.p, a.bytes, b->p, b->bytes),
                   "precondition_embedding: what is written overlaps another array");
  }
  char* ws = reinterpret_cast<char*>(
      (reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
  EmbedStep e = {};
  e.G = G_inv;
  e.A = A;
  e.damping = damping;
  e.grad = grad;
  e.kf = kf;
  e.param = param;
  e.mom = mom;
  e.lr = lr;
  e.momentum = momentum;
  e.vocab = (int)vocab;
  e.width = width;
  e.vec = (width & 3) == 0 &&
          ((reinterpret_cast<uintptr_t>(G_inv) | reinterpret_cast<uintptr_t>(grad) |
            reinterpret_cast<uintptr_t>(kf) | reinterpret_cast<uintptr_t>(param) |
            reinterpret_cast<uintptr_t>(mom)) & 15) == 0;
  const uintptr_t at = reinterpret_cast<uintptr_t>(kf);
  e.even = param == nullptr || (((at - reinterpret_cast<uintptr_t>(param)) |
                                 (at - reinterpret_cast<uintptr_t>(mom))) & 15) == 0;
  lay_out(vocab, width, ws, &e);
  cudaStream_t st = (cudaStream_t)stream;
  KFAC_CUDA(cudaMemsetAsync(e.count, 0, sizeof(int), st));
  const long long rows = vocab + width;
  embed_rows_kernel<<<(unsigned)std::min<long long>(parts_of(rows, kWarps),
                                                    (long long)sm_count() * 8),
                      kThreads, 0, st>>>(e);
  KFAC_LAUNCH_CHECK("embed_rows_kernel");
  PlaneLaunch<1> l;
  l.n = 1;
  PlaneFields& g = l.p[0].f;
  g = {};
  g.M = (int)vocab;
  g.N = g.K = width;
  if ((rc = plane_map(&l.p[0].ma, e.rows, (int)vocab, width, false)) != KFAC_OK ||
      (rc = plane_map(&l.p[0].mb, e.g, width, width, false)) != KFAC_OK)
    return rc;
  l.rows = e.count;
  rc = plane_launch("embed products", l, EpiEmbed{e}, true, st);
  if (rc != KFAC_OK || param == nullptr) return rc;
  return launch_behind("embed_update_kernel", true, embed_update_kernel,
                       (int)std::min<long long>(parts_of(vocab, kWarps),
                                                (long long)sm_count() * 8),
                       kThreads, 0, st, e);
}
