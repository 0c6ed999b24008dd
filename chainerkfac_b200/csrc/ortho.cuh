// What the two files of the orthogonalised updates share.
#pragma once

#include "common.cuh"

namespace kfac {

// Powers of two that X and A, B are held times (ortho.cu).
constexpr int kXExp = 13, kAExp = 12;
constexpr int kStepsMax = 64;

// Sides of the matrices that one block orthogonalises, the long side of those that a
// cluster of blocks does, and its part in a block (ortho_small.cu).
constexpr int kSmallShort = 128, kSmallLong = 256;
constexpr int kSmallShare = 192, kSmallClusterLong = 16 * kSmallShare;
constexpr int kSmallJobs = 64;

struct SmallJob {
  const void* x;
  void* dst;               // or null
  void* param;             // or null
  int rows, cols;
  float scale;
};

struct SmallLaunch {
  SmallJob j[kSmallJobs];
  int n, steps;
  int blocks;              // that share a matrix
  double eps;
  float keep, lr;
  float coefficients[3 * kStepsMax];
};
static_assert(sizeof(SmallLaunch) <= 4000, "kernel argument space");

int launch_ortho_small(SmallLaunch& l, int dtype, cudaStream_t st);

}  // namespace kfac
