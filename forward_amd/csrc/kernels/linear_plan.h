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
  int32_t whole_steps, tail;  // t as steps of a tile's depth and the elements that are left (`tail_of`)
  int32_t steps_per_split;    // of whole_steps (+ 1 for the tail) that one split walks
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
  void* dz;        // nullable; lines of ld_dz elements, zeros past n
  float* part;     // nullable: [gridDim.y][n] column sums of fp32 dz, before its rounding
  int64_t m;
  int32_t n, ld_dz;
  int32_t act;
};

// The tiles there are; `offered` in linear.hip says where.  The first three are the eight-wave kernel of 16-bit operands
// (product_turns_kernel), the others product_kernel with one shape of waves, step and buffers or another.  kFew:
// product_few_kernel, at most kFewRows rows of x.
enum TileKind {
  k256x256, k256x128, k128x128Turns, k64x64Alone, k128x128, k64x64, k64x32, k48x48, k48x32, k32x32Deep, k32x32, kTileKinds,
  kFew = kTileKinds
};
constexpr int kFewRows = 32;
struct TileShape {
  int ti, tj;
};
constexpr TileShape kTiles[kTileKinds] = {{256, 256}, {256, 128}, {128, 128}, {64, 64}, {128, 128}, {64, 64},
                                          {64, 32},   {48, 48},   {48, 32},   {32, 32}, {32, 32}};

// Bytes of t in a step.  The smallest tiles have the least to do between two barriers: operands straight from memory, which
// need no registers on the way, take 512 (fp16 512 x 1024 x 4096: 10.5 us, with 256 11.8).  So does k64x64Alone: a wave
// then multiplies all of the tile, which halves what it reads of it (bf16 1024 x 1024 x 4096, b across: 22 us, 26 with
// three buffers of 256); but 16-bit operands along t are better off with three buffers (15 us, 19).
inline int step_bytes(TileKind kind, int layouts, int elem, bool direct) {
  if (kind <= k128x128Turns || kind == k128x128) return 128;
  if (kind == k64x64Alone) return layouts == 0 && elem == 2 ? 256 : 512;
  if (kind == k64x32) return elem == 2 && direct ? 512 : 256;
  return kind == k48x48 || kind == k48x32 || kind == k32x32Deep ? 512 : 256;
}

struct Plan {
  TileKind tile;
  int splits, whole_steps, tail, steps_per_split;
  double us;  // estimate
};

// Both products of a gradient, unsplit and in tiles of one size, and the sums of its columns.
struct Gradients {
  Product x, w;
  int32_t blocks_x, blocks_w;
  TileKind tile;      // k64x64 or k32x32
  float* dbias;       // nullable
  const float* part;  // its partials [parts][n], or
  const void* dy;     // without partials, dy itself [parts][n]
  int64_t parts;
  int32_t n;
};

// Copies of up to two matrices with lines of `ld_out` elements, a multiple of 8, zeros past the `ld` of the source.
struct Widen {
  const void* in[2];
  void* out[2];
  int64_t lines[2];
  int32_t ld, ld_out;
};

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Operands that go from memory straight to LDS: 16-byte loads need 4-byte aligned lines, offsets are 31 bits.
inline bool direct_ok(const void* p, int64_t ld, int elem) {
  return reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld * elem % 4 == 0 && ld >= 8 && ld * elem <= (int64_t)1 << 22;
}

// How the end of t is loaded.  kWhole: every chunk that begins inside t is loaded whole, the last step like the others
// (t is a multiple of a chunk, or the lines are zeros from its end to the chunk's).  kTail: the elements past the last
// whole step go through registers.  kTailLine: so does at least the matrix's last line, because rows across t end
// inside a chunk and a line's last chunk reaches into the line behind it.
enum End { kWhole, kTail, kTailLine };

inline void tail_of(int nt, int depth, End end, int& whole, int& tail) {
  whole = end == kWhole ? ceil_div(nt, depth) : nt / depth;
  tail = end == kWhole ? 0 : nt % depth;
  if (end == kTailLine && tail == 0 && whole > 0) {
    --whole;
    tail = depth;
  }
}

// Run P as planned (with the finishing launch where t is split) / dz and its column sums, in elements of one type.
// layouts: 0 both along t, 1 a along and b across, 2 both across.
int run_product_f16(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream);
int run_product_bf16(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream);
int run_product_f32(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream);
int run_gradients_f16(const Gradients& G, bool direct, hipStream_t stream);
int run_gradients_bf16(const Gradients& G, bool direct, hipStream_t stream);
int run_gradients_f32(const Gradients& G, bool direct, hipStream_t stream);
int run_widen(const Widen& W, hipStream_t stream);  // 16-bit elements of either type
int run_slope_f16(const Slope& S, int parts, hipStream_t stream);
int run_slope_bf16(const Slope& S, int parts, hipStream_t stream);
int run_slope_f32(const Slope& S, int parts, hipStream_t stream);

}  // namespace fwdmi
