// What the linear launchers hand to their kernels and how they choose tiles and splits; compiled into one object per
// element type (linear_f16.hip, linear_bf16.hip, linear_f32.hip) and used by the entry points in linear.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../common.h"

namespace fwdmi {

enum Layout { kAlong = 0, kAcross = 1 };

struct Product {
  const void* a;  // kAlong: A(i, t) = a[i * lda + t]; kAcross: a[t * lda + i]
  const void* b;
  int64_t lda, ldb;
  int32_t ni, nj, nt;
  int32_t steps_per_split;  // steps of 128 bytes that one of gridDim.y splits walks
  float* partial;           // not null: C goes there unfinished, [split][ni][nj]
  void* c;                  // [ni, nj]
  void* preact;             // nullable
  const float* bias;        // [nj], nullable
  const void* residual;     // [ni, nj], nullable
  int32_t act;
  int32_t tiles_i, tiles_j;
};

// dz = dy * act'(z) and its column sums.
struct Slope {
  const void* dy;
  const void* z;   // nullable: dz = dy, only summed
  void* dz;
  float* part;     // nullable: [gridDim.y][n] column sums of fp32 dz, before its rounding
  int64_t m;
  int32_t n;
  int32_t act;
};

constexpr int kStepBytes = 128;  // of t that a step covers

enum TileKind { kBig = 0, kMid = 1, kSmall = 2 };
struct Plan {
  TileKind tile;
  int ti, tj;
  int splits, steps_per_split;
};

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Lines that are whole 16-byte chunks from a 16-byte boundary on, within a buffer load's 31-bit offsets.
inline bool direct_ok(const void* p, int64_t ld, int elem, int extent_along) {
  const int chunk = 16 / elem;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % chunk == 0 && extent_along % chunk == 0 &&
         ld * elem <= (int64_t)1 << 22;
}

// Run P as planned (with the finishing launch where t is split) / dz and its column sums, in elements of one type.
// layouts: 0 both along t, 1 a along and b across, 2 both across.
int run_product_f16(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream);
int run_product_bf16(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream);
int run_product_f32(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream);
int run_slope_f16(const Slope& S, int parts, hipStream_t stream);
int run_slope_bf16(const Slope& S, int parts, hipStream_t stream);
int run_slope_f32(const Slope& S, int parts, hipStream_t stream);

}  // namespace fwdmi
