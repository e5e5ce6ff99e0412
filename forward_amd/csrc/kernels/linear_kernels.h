// The linear layer on gfx950's matrix cores: a product with bias, activation and residual in its epilogue, and its
// gradient.
//
//   z = x w^T + b,  y = act(z) (+ residual)              x [m, k], w [n, k], y [m, n]
//   dz = dy * act'(z),  dx = dz w,  dw = dz^T x,  db = sum of dz over the rows
//
// One kernel does the three products: C(i, j) = sum over t of A(i, t) B(j, t) with either operand stored along t
// (kAlong: x and w of the forward product, dz of dx) or across it (kAcross: w of dx, both operands of dw).  A
// workgroup owns a TI x TJ tile of C and walks t in steps of 128 bytes; two LDS buffers, the next step's loads in
// flight while this one is multiplied, one barrier a step.  Sums are fp32 (the accumulators of the matrix cores).
//
// LDS holds a tile in 16-byte chunks, XOR-permuted so that the reads of a fragment spread over all banks:
//   kAlong   [row][128 bytes of t], chunk c of row r at c ^ (r & 7): a fragment is one ds_read_b128 a lane;
//   kAcross  [t][rows], the 32-byte (fp32: 64-byte) unit u of line t at u ^ f(t): 16-bit fragments are read
//            transposed (ds_read_b64_tr_b16), fp32 ones element by element.
// Operands whose lines are whole 16-byte chunks go from memory straight to LDS (buffer loads, whose range check
// supplies the zeros past the end of t); any other size or alignment passes through registers.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "linear_plan.h"
#include "slice.h"

namespace fwdmi {
namespace {

typedef float F4 __attribute__((ext_vector_type(4)));
typedef short S4 __attribute__((ext_vector_type(4)));
#define FWDMI_LDS __attribute__((address_space(3)))

// ---- activations ------------------------------------------------------------------------------------------------

__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// Phi(x), the normal distribution function: 1 - q(x) or q(|x|) with q the upper tail.  16-bit results take the
// tail from Abramowitz and Stegun 7.1.26 (absolute error of erf at most 1.5e-7), fp32 results from erfc itself.
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float x) {
  if (EXACT) return 0.5f * erfcf(-0.70710678118654752f * x);
  const float u = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, u, 1.0f));
  float p = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  p = __builtin_fmaf(t, p, 1.421413741f);
  p = __builtin_fmaf(t, p, -0.284496736f);
  p = __builtin_fmaf(t, p, 0.254829592f);
  const float q = 0.5f * p * t * exp_(-u * u);
  return x < 0.0f ? q : 1.0f - q;
}
// 1 / (1 + e^-x); e^-x overflows to infinity and the quotient to 0, as the limit is.
__device__ __forceinline__ float logistic(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_(-x)); }

constexpr float kTanhIn = 1.59576912160573071f;  // 2 sqrt(2 / pi): (1 + tanh(u)) / 2 = logistic(2 u)

template <int ACT, bool EXACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == FWDMI_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
  if (ACT == FWDMI_ACT_GELU) return z * normal_cdf<EXACT>(z);
  if (ACT == FWDMI_ACT_GELU_TANH) return z * logistic(kTanhIn * __builtin_fmaf(0.044715f * z, z * z, z));
  if (ACT == FWDMI_ACT_SILU) return z * logistic(z);
  return z;
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == FWDMI_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;
  if (ACT == FWDMI_ACT_GELU)
    return __builtin_fmaf(z * 0.39894228040143268f, exp_(-0.5f * z * z), normal_cdf<EXACT>(z));
  if (ACT == FWDMI_ACT_GELU_TANH) {
    const float p = logistic(kTanhIn * __builtin_fmaf(0.044715f * z, z * z, z));
    return __builtin_fmaf(z * p * (1.0f - p) * kTanhIn, __builtin_fmaf(0.134145f * z, z, 1.0f), p);
  }
  if (ACT == FWDMI_ACT_SILU) {
    const float p = logistic(z);
    return p * __builtin_fmaf(z, 1.0f - p, 1.0f);
  }
  return 1.0f;
}
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case FWDMI_ACT_RELU: f(std::integral_constant<int, FWDMI_ACT_RELU>{}); break;
    case FWDMI_ACT_GELU: f(std::integral_constant<int, FWDMI_ACT_GELU>{}); break;
    case FWDMI_ACT_GELU_TANH: f(std::integral_constant<int, FWDMI_ACT_GELU_TANH>{}); break;
    case FWDMI_ACT_SILU: f(std::integral_constant<int, FWDMI_ACT_SILU>{}); break;
    default: f(std::integral_constant<int, FWDMI_ACT_NONE>{}); break;
  }
}

// y = act(z) + residual, z = acc + bias, of eight neighbours of one row (columns j .. j + 7, those below nj exist).
template <typename T, int ACT>
__device__ __forceinline__ void finish(const Product& P, int64_t i, int j, const float (&acc)[8]) {
  const int64_t at = i * P.nj + j;
  const int live = min(P.nj - j, 8);
  Pack<T, 8> y, z, r{};
  float b[8] = {};
  if (live == 8) {
    if (P.bias) {
      const Pack<float, 4> lo = load_slice<float, 4>(gconst<float>(P.bias) + j);
      const Pack<float, 4> hi = load_slice<float, 4>(gconst<float>(P.bias) + j + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        b[e] = lo.v[e];
        b[e + 4] = hi.v[e];
      }
    }
    if (P.residual) r = load_slice<T, 8>(gconst<T>(P.residual) + at);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < live) {
        if (P.bias) b[e] = gconst<float>(P.bias)[j + e];
        if (P.residual) r.v[e] = gconst<T>(P.residual)[at + e];
      }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float s = acc[e] + b[e];
    z.v[e] = (T)s;
    y.v[e] = (T)(activate<ACT, sizeof(T) == 4>(s) + (float)r.v[e]);
  }
  if (live == 8) {
    store_slice<T, 8>(gmut<T>(P.c) + at, y);
    if (P.preact) store_slice<T, 8>(gmut<T>(P.preact) + at, z);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < live) {
        gmut<T>(P.c)[at + e] = y.v[e];
        if (P.preact) gmut<T>(P.preact)[at + e] = z.v[e];
      }
  }
}

// ---- tiles --------------------------------------------------------------------------------------------------------

template <typename T>
constexpr int kStep = kStepBytes / (int)sizeof(T);  // elements of t a step covers
template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);

// Position of a tile's chunks: ROWS * 8 of them, in the order they lie in LDS.
template <typename T, int ROWS, int LAYOUT>
struct Tile {
  static constexpr int kBytes = ROWS * kStepBytes;
  static constexpr int kLine = LAYOUT == kAlong ? kStepBytes : ROWS * (int)sizeof(T);  // bytes of an LDS line
  static constexpr int kUnit = sizeof(T) == 2 ? 2 : 4;                                 // chunks of a kAcross unit
  static constexpr int kUnits = kLine / (16 * kUnit);
  // what XOR permutes the units of line t by; fragments read 16 lines at a time: the bits that differ among them
  __device__ static __forceinline__ int across(int t) {
    const int f = sizeof(T) == 2 ? (t & 3) | ((t >> 1) & 4) : (t >> 2) & 3;
    return f & (kUnits - 1);
  }
  // the line and the chunk of the line whose contents lie at chunk p
  __device__ static __forceinline__ void locate(int p, int& line, int& chunk) {
    constexpr int per = kLine / 16;
    line = p / per;
    const int c = p % per;
    if (LAYOUT == kAlong)
      chunk = c ^ (line & 7);
    else
      chunk = ((c / kUnit) ^ across(line)) * kUnit + c % kUnit;
  }
};

// Loads of one operand's tile: ROWS rows from row `row0`, steps from `step0` on, by NT threads.
template <typename T, int ROWS, int LAYOUT, int NT, bool DIRECT>
struct Loader {
  using Tl = Tile<T, ROWS, LAYOUT>;
  static constexpr int kLoads = ROWS * 8 / NT;
  static_assert(ROWS * 8 % NT == 0, "whole loads");
  const T FWDMI_GLOBAL* base;  // the tile's first element at step0
  int64_t ld, step_elems;
  int rows, t_left;  // rows of the tile that exist; elements of t from the present step on
  int line[kLoads], chunk[kLoads];
  uint32_t offset[kLoads];
  Pack<T, kChunk<T>> held[DIRECT ? 1 : kLoads];

  __device__ __forceinline__ Loader(const void* p, int64_t ld_, int row0, int n_rows, int nt, int step0) {
    ld = ld_;
    rows = min(n_rows - row0, ROWS);
    t_left = nt - step0 * kStep<T>;
    const int64_t t0 = (int64_t)step0 * kStep<T>;
    base = gconst<T>(p) + (LAYOUT == kAlong ? row0 * ld + t0 : t0 * ld + row0);
    step_elems = LAYOUT == kAlong ? kStep<T> : kStep<T> * ld;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      Tl::locate(i * NT + (int)threadIdx.x, line[i], chunk[i]);
      offset[i] = (uint32_t)(line[i] * (uint32_t)(ld * sizeof(T)) + chunk[i] * 16);
    }
  }

  // DIRECT: issues the loads of the present step into `lds`; otherwise into registers (`drop` stores them).
  __device__ __forceinline__ void load(char* lds) {
    if constexpr (DIRECT) {
      // bytes from `base` to the end of what the tile may read; past it buffer loads give zeros
      const uint32_t lines = LAYOUT == kAlong ? rows : min(t_left, kStep<T>);
      const uint32_t last = LAYOUT == kAlong ? t_left : rows;
      const uint32_t bytes = ((lines - 1) * (uint32_t)ld + last) * (uint32_t)sizeof(T);
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
      const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        uint32_t at = offset[i];
        // a chunk of a row past the end of t would be the next row's beginning
        if (LAYOUT == kAlong && chunk[i] * kChunk<T> >= t_left) at = 0x80000000u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (FWDMI_LDS void*)(lds + (i * NT + wave * 64) * 16), 16, (int)at, 0,
                                                 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = LAYOUT == kAlong ? line[i] : chunk[i] * kChunk<T>;
        const int t = LAYOUT == kAlong ? chunk[i] * kChunk<T> : line[i];
        const T FWDMI_GLOBAL* const at = base + (int64_t)line[i] * ld + chunk[i] * kChunk<T>;
        const int n = r < rows && t < t_left ? (LAYOUT == kAlong ? t_left - t : rows - r) : 0;  // elements that exist
        if (n >= kChunk<T>) {
          held[i] = load_slice<T, kChunk<T>>(at);
        } else {
#pragma unroll
          for (int e = 0; e < kChunk<T>; ++e) held[i].v[e] = e < n ? at[e] : (T)0.0f;
        }
      }
    }
    base += step_elems;
    t_left -= kStep<T>;
  }
  __device__ __forceinline__ void drop(char* lds) {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        *reinterpret_cast<Pack<T, kChunk<T>>*>(lds + (i * NT + (int)threadIdx.x) * 16) = held[i];
    }
  }
};

// 16 rows x 16 bytes of t per lane quarter: what a lane feeds to one (16-bit) or four (fp32) matrix instructions.
template <typename T>
struct Frag {
  Pack<T, kChunk<T>> v;
};

// Reads the fragments of FR blocks of 16 rows from `row0` (a multiple of 16) on.
template <typename T, int ROWS, int LAYOUT, int FR>
struct Reader {
  using Tl = Tile<T, ROWS, LAYOUT>;
  int at[LAYOUT == kAlong ? 1 : FR];
  int half;
  __device__ __forceinline__ explicit Reader(int row0) {
    const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    half = 0;
    if constexpr (LAYOUT == kAlong) {
      at[0] = (row0 + j) * kStepBytes + ((g ^ (j & 7)) << 4);  // (row & 7 == j & 7); the second half flips bit 2
      half = ((g ^ (j & 7)) & 4) ? -64 : 64;
    } else if constexpr (sizeof(T) == 2) {
      const int t = g * 8 + (j >> 2);
#pragma unroll
      for (int f = 0; f < FR; ++f) at[f] = t * Tl::kLine + ((row0 / 16 + f) ^ Tl::across(t)) * 32 + (j & 3) * 8;
    } else {
#pragma unroll
      for (int f = 0; f < FR; ++f) at[f] = g * 4 * Tl::kLine + ((row0 / 16 + f) ^ Tl::across(g * 4)) * 64 + j * 4;
    }
  }
  // half h (of 64 bytes of t) of the step
  __device__ __forceinline__ void read(const char* lds, int h, Frag<T> (&out)[FR]) const {
#pragma unroll
    for (int f = 0; f < FR; ++f) {
      if constexpr (LAYOUT == kAlong) {
        out[f].v = *reinterpret_cast<const Pack<T, kChunk<T>>*>(lds + at[0] + h * half + f * 16 * kStepBytes);
      } else if constexpr (sizeof(T) == 2) {
        const char* const p = lds + at[f] + h * 32 * Tl::kLine;
        const S4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FWDMI_LDS S4*)(p));
        const S4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FWDMI_LDS S4*)(p + 4 * Tl::kLine));
        __builtin_memcpy(&out[f].v.v[0], &lo, 8);
        __builtin_memcpy(&out[f].v.v[4], &hi, 8);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          out[f].v.v[e] = *reinterpret_cast<const T*>(lds + at[f] + (h * 16 + e) * Tl::kLine);
      }
    }
  }
};

// acc(j block, i block) += B A^T: a lane holds four neighbouring j of one i.
template <typename T>
__device__ __forceinline__ F4 multiply(const Frag<T>& b, const Frag<T>& a, F4 acc) {
  if constexpr (std::is_same<T, _Float16>::value) {
    typedef _Float16 V __attribute__((ext_vector_type(8)));
    V vb, va;
    __builtin_memcpy(&vb, &b, 16);
    __builtin_memcpy(&va, &a, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, va, acc, 0, 0, 0);
  } else if constexpr (std::is_same<T, __bf16>::value) {
    typedef __bf16 V __attribute__((ext_vector_type(8)));
    V vb, va;
    __builtin_memcpy(&vb, &b, 16);
    __builtin_memcpy(&va, &a, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, va, acc, 0, 0, 0);
  } else {
    // element e of the four lane quarters is one step of four t: any order of t will do that both operands share
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(b.v.v[e], a.v.v[e], acc, 0, 0, 0);
    return acc;
  }
}

template <typename T, int LA, int LB, int TI, int TJ, int WI, int WJ, bool DIRECT>
__global__ __launch_bounds__(64 * WI * WJ) void product_kernel(const Product P) {
  constexpr int kNT = 64 * WI * WJ;
  constexpr int kFI = TI / WI / 16, kFJ = TJ / WJ / 16;
  using TileA = Tile<T, TI, LA>;
  using TileB = Tile<T, TJ, LB>;
  constexpr int kBuffer = TileA::kBytes + TileB::kBytes;  // one step of both operands
  __shared__ __attribute__((aligned(1024))) char s_tile[2 * kBuffer];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int ti = (int)(blockIdx.x % P.tiles_i), tj = (int)(blockIdx.x / P.tiles_i);
  const int i0 = ti * TI, j0 = tj * TJ;
  const int wi = wave % WI * (TI / WI), wj = wave / WI * (TJ / WJ);

  const int all = (P.nt + kStep<T> - 1) / kStep<T>;
  const int step0 = (int)blockIdx.y * P.steps_per_split;
  const int steps = min(all - step0, P.steps_per_split);

  F4 acc[kFJ][kFI];
#pragma unroll
  for (int j = 0; j < kFJ; ++j)
#pragma unroll
    for (int i = 0; i < kFI; ++i) acc[j][i] = F4{0.0f, 0.0f, 0.0f, 0.0f};

  if (steps > 0) {
    Loader<T, TI, LA, kNT, DIRECT> la(P.a, P.lda, i0, P.ni, P.nt, step0);
    Loader<T, TJ, LB, kNT, DIRECT> lb(P.b, P.ldb, j0, P.nj, P.nt, step0);
    const Reader<T, TI, LA, kFI> ra(wi);
    const Reader<T, TJ, LB, kFJ> rb(wj);
    la.load(s_tile);
    lb.load(s_tile + TileA::kBytes);
    la.drop(s_tile);
    lb.drop(s_tile + TileA::kBytes);
    for (int s = 0; s < steps; ++s) {
      char* const now = s_tile + (s & 1) * kBuffer;
      char* const next = s_tile + (~s & 1) * kBuffer;
      __syncthreads();  // this step's tiles are in LDS, and the other buffers have been read
      if (s + 1 < steps) {
        la.load(next);
        lb.load(next + TileA::kBytes);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        Frag<T> fa[kFI], fb[kFJ];
        ra.read(now, h, fa);
        rb.read(now + TileA::kBytes, h, fb);
#pragma unroll
        for (int j = 0; j < kFJ; ++j)
#pragma unroll
          for (int i = 0; i < kFI; ++i) acc[j][i] = multiply<T>(fb[j], fa[i], acc[j][i]);
      }
      if (s + 1 < steps) {
        la.drop(next);
        lb.drop(next + TileA::kBytes);
      }
    }
  }

  // The tile leaves through LDS, as much of it at a time as the buffers hold, so that every row is read back and
  // stored in whole 16-byte slices by neighbouring lanes.  16-byte chunk c of row r lies at c ^ (r & 15).
  constexpr int kPhases = std::max(1, TI * TJ * 4 / (2 * kBuffer));
  constexpr int kFP = kFI / kPhases;                // fragments of i a wave leaves per phase
  constexpr int kRowsPhase = TI / kPhases;          // rows of all waves per phase
  constexpr int kRowsWave = kRowsPhase / WI;
  float* const s_out = reinterpret_cast<float*>(s_tile);
  const int r_lane = wave % WI * kRowsWave + (lane & 15);
  for (int phase = 0; phase < kPhases; ++phase) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kPhases; ++p)
      if (p == phase) {
#pragma unroll
        for (int i = 0; i < kFP; ++i)
#pragma unroll
          for (int j = 0; j < kFJ; ++j) {
            const int chunk = ((wj + j * 16) / 4 + (lane >> 4)) ^ (lane & 15);
            *reinterpret_cast<F4*>(s_out + (r_lane + i * 16) * TJ + chunk * 4) = acc[j][p * kFP + i];
          }
      }
    __syncthreads();
    auto leave = [&](auto&& f) {
#pragma unroll 1
      for (int q = threadIdx.x; q < kRowsPhase * TJ / 8; q += kNT) {
        const int row = q / (TJ / 8), c = q % (TJ / 8);
        const int i = i0 + row / kRowsWave * (TI / WI) + phase * kRowsWave + row % kRowsWave, j = j0 + c * 8;
        if (i >= P.ni || j >= P.nj) continue;
        const F4 lo = *reinterpret_cast<const F4*>(s_out + row * TJ + ((2 * c) ^ (row & 15)) * 4);
        const F4 hi = *reinterpret_cast<const F4*>(s_out + row * TJ + ((2 * c + 1) ^ (row & 15)) * 4);
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        f((int64_t)i, j, v);
      }
    };
    if (P.partial) {
      float FWDMI_GLOBAL* const out = gmut<float>(P.partial) + (int64_t)blockIdx.y * P.ni * P.nj;
      leave([&](int64_t i, int j, const float (&v)[8]) {
        float FWDMI_GLOBAL* const p = out + i * P.nj + j;
        if (j + 8 <= P.nj) {
          store_slice<float, 4>(p, Pack<float, 4>{v[0], v[1], v[2], v[3]});
          store_slice<float, 4>(p + 4, Pack<float, 4>{v[4], v[5], v[6], v[7]});
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (j + e < P.nj) p[e] = v[e];
        }
      });
    } else if constexpr (LA == kAlong && LB == kAlong) {
      with_act(P.act, [&](auto act) {
        leave([&](int64_t i, int j, const float (&v)[8]) { finish<T, decltype(act)::value>(P, i, j, v); });
      });
    } else {  // the gradient's products have no epilogue
      leave([&](int64_t i, int j, const float (&v)[8]) { finish<T, FWDMI_ACT_NONE>(P, i, j, v); });
    }
  }
}

// Adds the splits' partial products in split order and finishes them; eight neighbours of a row per lane.
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(const Product P, int splits) {
  const int per = (P.nj + 7) / 8;
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t i = q / per;
  if (i >= P.ni) return;
  const int j = (int)(q % per) * 8;
  const int64_t plane = (int64_t)P.ni * P.nj;
  const float FWDMI_GLOBAL* p = gconst<float>(P.partial) + i * P.nj + j;
  const int live = min(P.nj - j, 8);
  float acc[8] = {};
  for (int s = 0; s < splits; ++s, p += plane) {
    if (live == 8) {
      const Pack<float, 4> lo = load_slice<float, 4>(p), hi = load_slice<float, 4>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[e] += lo.v[e];
        acc[e + 4] += hi.v[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < live) acc[e] += p[e];
    }
  }
  with_act(P.act, [&](auto act) { finish<T, decltype(act)::value>(P, i, j, acc); });
}

// ---- dz = dy * act'(z) and its column sums -----------------------------------------------------------------------

// 512 columns (8 per lane) x every (4 gridDim.y)-th row per wave, the four waves' sums through LDS.
template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(const Slope S) {
  constexpr int kVec = 8;
  __shared__ float s_sum[4][64 * kVec];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x * 64 + lane) * kVec;
  const int live = min(max(S.n - c, 0), kVec);
  float sum[kVec] = {};
  with_act(S.act, [&](auto act) {
    if (live == 0) return;
    for (int64_t r = blockIdx.y * 4 + wave; r < S.m; r += 4 * gridDim.y) {
      const int64_t at = r * S.n + c;
      Pack<T, kVec> dy{}, z{};
      if (live == kVec) {
        dy = load_slice<T, kVec>(gconst<T>(S.dy) + at);
        if (S.z) z = load_slice<T, kVec>(gconst<T>(S.z) + at);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (e < live) {
            dy.v[e] = gconst<T>(S.dy)[at + e];
            if (S.z) z.v[e] = gconst<T>(S.z)[at + e];
          }
      }
      Pack<T, kVec> out;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        float v = (float)dy.v[e];
        if (decltype(act)::value != FWDMI_ACT_NONE) v *= slope<decltype(act)::value, sizeof(T) == 4>((float)z.v[e]);
        sum[e] += v;
        out.v[e] = (T)v;
      }
      if (S.dz) {
        if (live == kVec) {
          store_slice<T, kVec>(gmut<T>(S.dz) + at, out);
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (e < live) gmut<T>(S.dz)[at + e] = out.v[e];
        }
      }
    }
  });
  if (!S.part) return;
#pragma unroll
  for (int e = 0; e < kVec; ++e) s_sum[wave][lane * kVec + e] = sum[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * kVec; i += 256) {
    const int col = blockIdx.x * 64 * kVec + i;
    if (col < S.n) gmut<float>(S.part)[(int64_t)blockIdx.y * S.n + col] = ((s_sum[0][i] + s_sum[1][i]) + s_sum[2][i]) + s_sum[3][i];
  }
}

template <typename T, int LA, int LB, bool DIRECT>
int launch_product(Product& P, const Plan& plan, hipStream_t stream) {
  P.tiles_i = ceil_div(P.ni, plan.ti);
  P.tiles_j = ceil_div(P.nj, plan.tj);
  P.steps_per_split = plan.steps_per_split;
  const dim3 grid((unsigned)(P.tiles_i * P.tiles_j), (unsigned)plan.splits);
  if constexpr (sizeof(T) == 2 && DIRECT) {
    if (plan.tile == kBig) hipLaunchKernelGGL((product_kernel<T, LA, LB, 256, 256, 2, 4, true>), grid, dim3(512), 0, stream, P);
  }
  if (plan.tile == kMid) hipLaunchKernelGGL((product_kernel<T, LA, LB, 128, 128, 2, 2, DIRECT>), grid, dim3(256), 0, stream, P);
  if (plan.tile == kSmall) hipLaunchKernelGGL((product_kernel<T, LA, LB, 64, 64, 2, 2, DIRECT>), grid, dim3(256), 0, stream, P);
  FWDMI_HIP_CHECK(hipGetLastError());
  if (plan.splits > 1) {
    const int64_t octets = (int64_t)P.ni * ((P.nj + 7) / 8);
    hipLaunchKernelGGL((finish_kernel<T>), dim3((unsigned)ceil_div(octets, 256)), dim3(256), 0, stream, P, plan.splits);
    FWDMI_HIP_CHECK(hipGetLastError());
  }
  return FWDMI_OK;
}

template <typename T, bool DIRECT>
int launch_layouts(Product& P, int layouts, const Plan& plan, hipStream_t stream) {
  if (layouts == 0) return launch_product<T, kAlong, kAlong, DIRECT>(P, plan, stream);
  if (layouts == 1) return launch_product<T, kAlong, kAcross, DIRECT>(P, plan, stream);
  return launch_product<T, kAcross, kAcross, DIRECT>(P, plan, stream);
}
template <typename T>
int run_product(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream) {
  return direct ? launch_layouts<T, true>(P, layouts, plan, stream) : launch_layouts<T, false>(P, layouts, plan, stream);
}
template <typename T>
int run_slope(const Slope& S, int parts, hipStream_t stream) {
  const dim3 grid((unsigned)ceil_div(S.n, 512), (unsigned)parts);
  hipLaunchKernelGGL((slope_kernel<T>), grid, dim3(256), 0, stream, S);
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

}  // namespace
}  // namespace fwdmi
