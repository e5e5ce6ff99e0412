// The linear layer on gfx950's matrix cores: a product with bias, activation and residual in its epilogue, and its
// gradient.
//
//   z = x w^T + b,  y = act(z) (+ residual)              x [m, k], w [n, k], y [m, n]
//   dz = dy * act'(z),  dx = dz w,  dw = dz^T x,  db = sum of dz over the rows
//
// One kernel does the three products: C(i, j) = sum over t of A(i, t) B(j, t) with either operand stored along t
// (kAlong: x and w of the forward product, dz of dx) or across it (kAcross: w of dx, both operands of dw).  A
// workgroup owns a TI x TJ tile of C and walks t in steps of 128 to 512 bytes; two to four LDS buffers, the next
// steps' loads in flight while this one is multiplied.  Sums are fp32 (the accumulators of the matrix cores).
//
// LDS holds a tile in 16-byte chunks, XOR-permuted so that the reads of a fragment spread over all banks:
//   kAlong   [row][bytes of t of a step], chunk c of row r at c ^ (r & 7): a fragment is one ds_read_b128 a lane;
//   kAcross  [t][rows], the 32-byte (fp32: 64-byte) unit u of line t at u ^ f(t): 16-bit fragments are read
//            transposed (ds_read_b64_tr_b16), fp32 ones element by element.
// Operands whose lines are whole 4-byte words go from memory straight to LDS (buffer loads, whose range check
// supplies the zeros past the end of t); any other size or alignment passes through registers.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "linear_plan.h"
#include "slice.h"

namespace fwdmi {
namespace {

typedef float F4 __attribute__((ext_vector_type(4)));
typedef short S4 __attribute__((ext_vector_type(4)));
#define FWDMI_LDS __attribute__((address_space(3)))

// ---- activations ------------------------------------------------------------------------------------------------

__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// EXACT, for fp32 results: a rounding of an exponent's argument enters the result times the argument (silu(-16) was 16 units
// of 2^-24 off, gelu_tanh(-9) 200), so arguments are formed in 64 bits and go in as a sum of two floats.  16-bit results round
// by a thousand times more.
struct Two {
  float hi, lo;
  __device__ __forceinline__ explicit Two(double a) : hi((float)a), lo((float)(a - (double)(float)a)) {}
};
// e^-a for a >= 0 (2^-24 relative, a few units; from a = 200 on it is 0)
__device__ __forceinline__ float exp_minus(double a) {
  const Two t(fmin(a, 200.0));
  return expf(-t.hi) * (1.0f - t.lo);
}

// Phi(x), the normal distribution function: 1 - q(x) or q(|x|) with q the upper tail.  fp32 results take it from erfc itself,
// at the rounded argument and with the slope for the rest.  16-bit results take the tail from Abramowitz and Stegun 7.1.26
// (absolute error of erf at most 1.5e-7; of the tail's own value 0.05 % at x = -4, 0.16 % at -5, 0.4 % at -6, where bf16
// rounds by as much, 1 % at -8, 3.7 % at -13).
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float x) {
  if (EXACT) {
    const Two u(fmin(fmax((double)x * -0.70710678118654752440, -30.0), 30.0));
    return __builtin_fmaf(exp_(-u.hi * u.hi) * -0.56418958354775629f, u.lo, 0.5f * erfcf(u.hi));
  }
  const float u = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, u, 1.0f));
  float p = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  p = __builtin_fmaf(t, p, 1.421413741f);
  p = __builtin_fmaf(t, p, -0.284496736f);
  p = __builtin_fmaf(t, p, 0.254829592f);
  const float q = 0.5f * p * t * exp_(-u * u);
  return x < 0.0f ? q : 1.0f - q;
}
// The normal density times sqrt(2 pi).
template <bool EXACT>
__device__ __forceinline__ float bell(float x) {
  return EXACT ? exp_minus(0.5 * (double)x * (double)x) : exp_(-0.5f * x * x);
}

// p = 1 / (1 + e^-a) and 1 - p.
struct Logistic {
  float p, rest;
};
template <bool EXACT, typename A>
__device__ __forceinline__ Logistic logistic(A a) {
  if (EXACT) {  // neither cancels nor overflows; what is below 2^-126 is 0, here as there (silu(-100) is -0)
    const float e = exp_minus(fabs((double)a)), t = e < 0x1p-126f ? 0.0f : e, r = __builtin_amdgcn_rcpf(1.0f + t);
    return a < 0 ? Logistic{t * r, r} : Logistic{r, t * r};
  }
  // e^-a overflows to infinity and the quotient to 0, as the limit is
  const float p = __builtin_amdgcn_rcpf(1.0f + exp_(-(float)a));
  return Logistic{p, 1.0f - p};
}

constexpr float kTanhIn = 1.59576912160573071f;  // 2 sqrt(2 / pi): (1 + tanh(u)) / 2 = logistic(2 u)
template <bool EXACT>
__device__ __forceinline__ Logistic gelu_tanh(float z) {
  if (EXACT) {
    const double d = z;
    return logistic<true>(1.59576912160573071 * d * __builtin_fma(0.044715 * d, d, 1.0));
  }
  return logistic<false>(kTanhIn * __builtin_fmaf(0.044715f * z, z * z, z));
}

template <int ACT, bool EXACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == FWDMI_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
  if (ACT == FWDMI_ACT_GELU) return z * normal_cdf<EXACT>(z);
  if (ACT == FWDMI_ACT_GELU_TANH) return z * gelu_tanh<EXACT>(z).p;
  if (ACT == FWDMI_ACT_SILU) return z * logistic<EXACT>(z).p;
  return z;
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == FWDMI_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;
  if (ACT == FWDMI_ACT_GELU) return __builtin_fmaf(z * 0.39894228040143268f, bell<EXACT>(z), normal_cdf<EXACT>(z));
  if (ACT == FWDMI_ACT_GELU_TANH) {
    const Logistic l = gelu_tanh<EXACT>(z);
    const float zz = fminf(z * z, 1e30f);  // (where it would overflow p (1 - p) is zero; NaN comes back with p)
    return __builtin_fmaf(z * l.p * l.rest * kTanhIn, __builtin_fmaf(0.134145f, zz, 1.0f), l.p);
  }
  if (ACT == FWDMI_ACT_SILU) {
    const Logistic l = logistic<EXACT>(z);
    return l.p * __builtin_fmaf(z, l.rest, 1.0f);
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

template <int N>
__device__ __forceinline__ void load_bias(const Product& P, int j, float (&b)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) b[e] = 0.0f;
  if (!P.bias) return;
  if (j + N <= P.nj) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const Pack<float, 4> v = load_slice<float, 4>(gconst<float>(P.bias) + j + q * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[q * 4 + e] = v.v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (j + e < P.nj) b[e] = gconst<float>(P.bias)[j + e];
  }
}

// y = act(z) + residual, z = acc + bias, of N neighbours of one row: those of columns j .. j + N - 1 that are below nj.
template <typename T, int ACT, int N>
__device__ __forceinline__ void finish(const Product& P, int64_t i, int j, const float (&acc)[N], const float (&b)[N]) {
  const int64_t at = i * P.nj + j;
  const int live = min(P.nj - j, N);
  Pack<T, N> y, z, r{};
  if (P.residual) {
    if (live == N) {
      r = load_slice<T, N>(gconst<T>(P.residual) + at);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < live) r.v[e] = gconst<T>(P.residual)[at + e];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float s = acc[e] + b[e];
    z.v[e] = (T)s;
    y.v[e] = (T)(activate<ACT, sizeof(T) == 4>(s) + (float)r.v[e]);
  }
  if (live == N) {
    store_slice<T, N>(gmut<T>(P.c) + at, y);
    if (P.preact) store_slice<T, N>(gmut<T>(P.preact) + at, z);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < live) {
        gmut<T>(P.c)[at + e] = y.v[e];
        if (P.preact) gmut<T>(P.preact)[at + e] = z.v[e];
      }
  }
}

// ---- tiles --------------------------------------------------------------------------------------------------------

template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);

// Position of a tile's chunks in LDS: ROWS rows by STEP bytes of t.
template <typename T, int ROWS, int LAYOUT, int STEP>
struct Tile {
  static constexpr int kBytes = ROWS * STEP;
  static constexpr int kT = STEP / (int)sizeof(T);                            // elements of t
  static constexpr int kLine = LAYOUT == kAlong ? STEP : ROWS * (int)sizeof(T);  // bytes of an LDS line
  static constexpr int kUnit = sizeof(T) == 2 ? 2 : 4;                        // chunks of a kAcross unit
  static constexpr int kUnits = kLine / (16 * kUnit);
  // what XOR permutes the chunks of row r by: 16 rows, eight of one chunk and eight of its neighbour, fill 256 bytes
  __device__ static __forceinline__ int along(int r) { return r & (STEP >= 256 ? 15 : 7); }
  // what XOR permutes the units of line t by.  16-bit fragments read lines 0 .. 3 and 8 .. 11 at a time, which fill 256
  // bytes: lines of 256 bytes and more differ by three bits, two lines of 128 to 256 bytes by two, four by one.
  __device__ static __forceinline__ int across(int t) {
    if (sizeof(T) == 4) return ((t >> 2) & 3) & (kUnits - 1);
    return kUnits >= 8 ? (t & 3) | ((t >> 1) & 4) : kUnits == 4 ? ((t >> 1) & 1) | ((t >> 2) & 2) : (t >> 3) & (kUnits - 1);
  }
  // the line and the chunk of the line whose contents lie at chunk p
  __device__ static __forceinline__ void locate(int p, int& line, int& chunk) {
    constexpr int per = kLine / 16;
    line = p / per;
    const int c = p % per;
    if (LAYOUT == kAlong)
      chunk = c ^ along(line);
    else
      chunk = ((c / kUnit) ^ across(line)) * kUnit + c % kUnit;
  }
};

// Loads of one operand's tile by NT threads: ROWS rows from row `row0` on, steps of t from `step0` on.
// DIRECT: memory to LDS, `left` steps and then nothing; else through registers, two sets of them.
template <typename T, int ROWS, int LAYOUT, int STEP, int NT, bool DIRECT>
struct Loader {
  using Tl = Tile<T, ROWS, LAYOUT, STEP>;
  static constexpr int kLoads = Tl::kBytes / 16 / NT;
  static_assert(Tl::kBytes % (16 * NT) == 0, "whole loads");
  const T FWDMI_GLOBAL* base;  // the tile's first element in the present step
  int64_t ld, step_elems;
  int rows, left;  // rows of the tile that exist; steps left
  int t_left;      // elements of t left (of the whole matrix, DIRECT, or of the split)
  int partial;     // DIRECT: the value of `left` at which a step is the matrix's last and partial, 0 for never
  uint32_t bytes;  // DIRECT: from `base` to the end of what a step may read
  int line[kLoads], chunk[kLoads];
  uint32_t offset[DIRECT ? kLoads : 1];
  Pack<T, kChunk<T>> held[DIRECT ? 1 : 2][DIRECT ? 1 : kLoads];

  __device__ __forceinline__ Loader(const void* p, int64_t ld_, int row0, int n_rows, int step0, int left_, int t_left_) {
    ld = ld_;
    rows = min(n_rows - row0, ROWS);
    left = left_;
    t_left = t_left_;
    const int64_t t0 = (int64_t)step0 * Tl::kT;
    base = gconst<T>(p) + (LAYOUT == kAlong ? row0 * ld + t0 : t0 * ld + row0);
    step_elems = LAYOUT == kAlong ? Tl::kT : Tl::kT * ld;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      Tl::locate(i * NT + (int)threadIdx.x, line[i], chunk[i]);
      if (DIRECT) offset[i] = (uint32_t)(line[i] * (uint32_t)(ld * sizeof(T)) + chunk[i] * 16);
    }
    if (DIRECT) {
      bytes = readable(Tl::kT);
      partial = left * Tl::kT > t_left ? 1 : 0;
    }
  }

  // ---- DIRECT
  // Bytes from `base` to the end of what a step with t elements of t may read; past it buffer loads give zeros and touch
  // nothing.  (The last chunk of a line may reach past the rows or past t: into zeros, or into the next line, `tail_of`.)
  __device__ __forceinline__ uint32_t readable(int t) const {
    constexpr int kC = kChunk<T>;
    const uint32_t lines = LAYOUT == kAlong ? rows : t, last = ((LAYOUT == kAlong ? t : rows) + kC - 1) / kC * kC;
    return ((lines - 1) * (uint32_t)ld + last) * (uint32_t)sizeof(T);
  }
  __device__ __forceinline__ void load(char* lds) {
    // Few scalar instructions: a wave's loads wait for them at the head of every step.
    if (left == partial) {  // also past the end, where there is nothing to read
      bytes = left > 0 ? readable(t_left) : 0;
      if (LAYOUT == kAlong)  // a chunk past the end of t would be the next row's beginning
#pragma unroll
        for (int i = 0; i < kLoads; ++i) offset[i] = chunk[i] * kChunk<T> < t_left ? offset[i] : 0x80000000u;
      partial = 0;
    }
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (FWDMI_LDS void*)(lds + (i * NT + wave * 64) * 16), 16,
                                               (int)offset[i], 0, 0, 0);
    base += step_elems;
    t_left -= Tl::kT;
    --left;
  }

  // ---- through registers
  // Chunk i of the step at `base` that has `t_left` elements of t, zeros where nothing exists.
  __device__ __forceinline__ Pack<T, kChunk<T>> some(const T FWDMI_GLOBAL* base, int i, int t_left) const {
    const int r = LAYOUT == kAlong ? line[i] : chunk[i] * kChunk<T>;
    const int t = LAYOUT == kAlong ? chunk[i] * kChunk<T> : line[i];
    const int n = r < rows && t < t_left ? (LAYOUT == kAlong ? t_left - t : rows - r) : 0;
    const T FWDMI_GLOBAL* const at = base + (n > 0 ? (int64_t)line[i] * ld + chunk[i] * kChunk<T> : 0);
    Pack<T, kChunk<T>> v;
    if (n >= kChunk<T>) {
      v = load_slice<T, kChunk<T>>(at);
    } else {
#pragma unroll
      for (int e = 0; e < kChunk<T>; ++e) v.v[e] = e < n ? at[e] : (T)0.0f;
    }
    return v;
  }
  __device__ __forceinline__ void put(char* lds, int i, const Pack<T, kChunk<T>>& v) const {
    *reinterpret_cast<Pack<T, kChunk<T>>*>(lds + (i * NT + (int)threadIdx.x) * 16) = v;
  }
  template <int SET>
  __device__ __forceinline__ void fetch() {
    // A step whose loads all lie inside the matrix takes them whole: rows past the tile's last repeat one (nobody
    // reads their products), a line's last chunk may reach up to a chunk less one element into the lines behind it.
    const bool whole = t_left >= Tl::kT && (LAYOUT == kAlong || rows % kChunk<T> == 0 ||
                                            (int64_t)(t_left - Tl::kT) * ld >= kChunk<T> - 1);
    if (whole) {
      const int most = LAYOUT == kAlong ? rows - 1 : (rows + kChunk<T> - 1) / kChunk<T> - 1;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int l = LAYOUT == kAlong ? min(line[i], most) : line[i], c = LAYOUT == kAlong ? chunk[i] : min(chunk[i], most);
        held[SET][i] = load_slice<T, kChunk<T>>(base + (int64_t)l * ld + c * kChunk<T>);
      }
    } else if (t_left > 0) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) held[SET][i] = some(base, i, t_left);
    }
    base += step_elems;
    t_left -= Tl::kT;
  }
  template <int SET>
  __device__ __forceinline__ void drop(char* lds) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) put(lds, i, held[SET][i]);
  }
  // The last, partial step of DIRECT loads, `steps` past `base`.
  __device__ __forceinline__ void tail(char* lds, int steps, int t_left) const {
    const T FWDMI_GLOBAL* const at = base + steps * step_elems;
    Pack<T, kChunk<T>> v[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = some(at, i, t_left);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) put(lds, i, v[i]);
  }
};

// 16 rows x 16 bytes of t per lane quarter: what a lane feeds to one (16-bit) or four (fp32) matrix instructions.
template <typename T>
struct Frag {
  Pack<T, kChunk<T>> v;
};

// Reads the fragments of FR blocks of 16 rows from `row0` (a multiple of 16) on.
template <typename T, int ROWS, int LAYOUT, int STEP, int FR>
struct Reader {
  using Tl = Tile<T, ROWS, LAYOUT, STEP>;
  int at[LAYOUT == kAlong ? 1 : FR];
  int half, quarter;
  __device__ __forceinline__ explicit Reader(int row0) {
    const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    half = quarter = 0;
    if constexpr (LAYOUT == kAlong) {
      at[0] = (row0 + j) * STEP + ((g ^ Tl::along(j)) << 4);  // (row0 is a multiple of 16)
      half = (g ^ Tl::along(j)) & 4;     // 64 bytes more flip bit 2 of the chunk,
      quarter = (g ^ Tl::along(j)) & 8;  // 128 bytes more bit 3
    } else if constexpr (sizeof(T) == 2) {
      const int t = g * 8 + (j >> 2);
#pragma unroll
      for (int f = 0; f < FR; ++f) at[f] = t * Tl::kLine + ((row0 / 16 + f) ^ Tl::across(t)) * 32 + (j & 3) * 8;
    } else {
#pragma unroll
      for (int f = 0; f < FR; ++f) at[f] = g * 4 * Tl::kLine + ((row0 / 16 + f) ^ Tl::across(g * 4)) * 64 + j * 4;
    }
  }
  // blocks FIRST .. FIRST + COUNT - 1 of half h (64 bytes of t) of the step
  template <int FIRST = 0, int COUNT = FR>
  __device__ __forceinline__ void read(const char* lds, int h, Frag<T> (&out)[COUNT]) const {
#pragma unroll
    for (int f = 0; f < COUNT; ++f) {
      if constexpr (LAYOUT == kAlong) {
        out[f].v = *reinterpret_cast<const Pack<T, kChunk<T>>*>(lds + at[0] + (h & 1 ? 64 - 32 * half : 0) +
                                                                  (h & 2 ? 128 - 32 * quarter : 0) + (h >> 2) * 256 +
                                                                  (FIRST + f) * 16 * STEP);
      } else if constexpr (sizeof(T) == 2) {
        const char* const p = lds + at[FIRST + f] + h * 32 * Tl::kLine;
        const S4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FWDMI_LDS S4*)(p));
        const S4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FWDMI_LDS S4*)(p + 4 * Tl::kLine));
        __builtin_memcpy(&out[f].v.v[0], &lo, 8);
        __builtin_memcpy(&out[f].v.v[4], &hi, 8);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          out[f].v.v[e] = *reinterpret_cast<const T*>(lds + at[FIRST + f] + (h * 16 + e) * Tl::kLine);
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

// All of a fragment row against all of a fragment column; fp32 goes through one step of t for every accumulator before the
// next, so that no instruction waits for the sum of the one before it.
template <typename T, int FI, int FJ>
__device__ __forceinline__ void multiply_all(const Frag<T> (&b)[FJ], const Frag<T> (&a)[FI], F4 (&acc)[FJ][FI]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
      for (int i = 0; i < FI; ++i) acc[j][i] = multiply<T>(b[j], a[i], acc[j][i]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int i = 0; i < FI; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j].v.v[e], a[i].v.v[e], acc[j][i], 0, 0, 0);
  }
}

// The steps of t that a split walks: whole ones from `first` on, and `tail` elements of a last one.
struct Steps {
  int first, whole, tail;
};
__device__ __forceinline__ Steps split_steps(const Product& P, int split) {
  const int first = split * P.steps_per_split, end = first + P.steps_per_split;
  const int whole = max(min(end, P.whole_steps) - first, 0);
  return Steps{first, whole, first <= P.whole_steps && end > P.whole_steps ? P.tail : 0};
}

// The immediate of s_waitcnt that waits until at most n vector memory operations are in flight (and for nothing else).
constexpr int wait_loads(int n) { return (n & 15) | (n >> 4) << 14 | 0x0f70; }

// The tile and split of workgroup b of `total`.  Workgroups go to the XCDs in turn, so the numbers are dealt out in eight runs
// of neighbours, one per XCD; a run stays in one split as long as it can and walks columns of at most kGroup tiles, so
// that the tiles an XCD works on at a time share their lines of A and B in its L2.
template <int TI, int TJ>
__device__ __forceinline__ int locate_tile(const Product& P, int b, int total, int& i0, int& j0) {
  const int tiles = P.tiles_i * P.tiles_j;
  const int xcd = b & 7, per = total >> 3, more = total & 7;
  const int n = xcd * per + min(xcd, more) + (b >> 3);
  const int split = n / tiles, m = n - split * tiles;
  constexpr int kGroup = TI > TJ ? 4 : 8;
  const int group = m / (kGroup * P.tiles_j), first = group * kGroup;
  const int height = min(P.tiles_i - first, kGroup), in = m - group * kGroup * P.tiles_j;
  i0 = (first + in % height) * TI;
  j0 = in / height * TJ;
  return split;
}

// The tile leaves through LDS, as much of it at a time as the buffers hold, so that every row is read back and stored
// in whole 16-byte slices by neighbouring lanes.  16-byte chunk c of row r lies at c ^ (r & 15).
template <typename T, int TI, int TJ, int WI, int WJ, int WK, int ROOM, bool EPILOGUE, int FI, int FJ>
__device__ __forceinline__ void leave_tile(const Product& P, const F4 (&acc)[FJ][FI], char* s_tile, int i0, int j0,
                                           int split) {
  constexpr int kNT = 64 * WI * WJ * WK;
  constexpr int kAllBytes = TI * TJ * 4 * WK;
  constexpr int kPhases = kAllBytes <= ROOM ? 1 : kAllBytes <= 2 * ROOM ? 2 : 4;
  static_assert(kAllBytes / kPhases <= ROOM && FI % kPhases == 0, "a part of the tile fits the buffers");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wj = wave / WI % WJ * (TJ / WJ);
  constexpr int kFP = FI / kPhases;                // fragments of i a wave leaves per phase
  constexpr int kRowsPhase = TI / kPhases;          // rows of all waves per phase
  constexpr int kRowsWave = kRowsPhase / WI;
  constexpr int kMix = ((TJ / 4 & -(TJ / 4)) < 16 ? TJ / 4 & -(TJ / 4) : 16) - 1;  // of a row's chunks, an even share
  constexpr int kSlab = kRowsPhase * TJ;            // elements of a wave group's part of the sum over t
  float* const s_out = reinterpret_cast<float*>(s_tile);
  float* const s_mine = s_out + wave / (WI * WJ) * kSlab;
  const int r_lane = wave % WI * kRowsWave + (lane & 15);
  for (int phase = 0; phase < kPhases; ++phase) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kPhases; ++p)
      if (p == phase) {
#pragma unroll
        for (int i = 0; i < kFP; ++i)
#pragma unroll
          for (int j = 0; j < FJ; ++j) {
            const int chunk = ((wj + j * 16) / 4 + (lane >> 4)) ^ (lane & kMix);
            *reinterpret_cast<F4*>(s_mine + (r_lane + i * 16) * TJ + chunk * 4) = acc[j][p * kFP + i];
          }
      }
    __syncthreads();
    auto leave = [&](auto&& f) {
#pragma unroll 1
      for (int q = threadIdx.x; q < kRowsPhase * TJ / 8; q += kNT) {
        const int row = q / (TJ / 8), c = q % (TJ / 8);
        const int i = i0 + row / kRowsWave * (TI / WI) + phase * kRowsWave + row % kRowsWave, j = j0 + c * 8;
        if (i >= P.ni || j >= P.nj) continue;
        F4 lo{0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
#pragma unroll
        for (int k = 0; k < WK; ++k) {
          lo += *reinterpret_cast<const F4*>(s_out + k * kSlab + row * TJ + ((2 * c) ^ (row & kMix)) * 4);
          hi += *reinterpret_cast<const F4*>(s_out + k * kSlab + row * TJ + ((2 * c + 1) ^ (row & kMix)) * 4);
        }
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        f((int64_t)i, j, v);
      }
    };
    if (P.partial) {
      float FWDMI_GLOBAL* const out = gmut<float>(P.partial) + (int64_t)split * P.ni * P.nj;
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
    } else if constexpr (EPILOGUE) {
      with_act(P.act, [&](auto act) {
        leave([&](int64_t i, int j, const float (&v)[8]) {
          float b[8];
          load_bias(P, j, b);
          finish<T, decltype(act)::value>(P, i, j, v, b);
        });
      });
    } else {  // the gradient's products have no epilogue
      leave([&](int64_t i, int j, const float (&v)[8]) {
        const float b[8] = {};
        finish<T, FWDMI_ACT_NONE>(P, i, j, v, b);
      });
    }
  }
}

// A tile of 16-bit results whose columns all exist leaves straight from the accumulators: no LDS, no barrier, and the two
// waves of a SIMD overlap each other's arithmetic and stores.  A lane holds four neighbouring columns of blocks 2 p and
// 2 p + 1; exchanges between the lane rows (16 lanes each) give it eight neighbouring columns of one block.
template <typename T, int TI, int TJ, int WI, int WJ, bool EPILOGUE, int FI, int FJ>
__device__ __forceinline__ void leave_registers(const Product& P, const F4 (&acc)[FJ][FI], int i0, int j0, int split) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int i_lane = i0 + wave % WI * (TI / WI) + (lane & 15);
  const int j_lane = j0 + wave / WI * (TJ / WJ) + (g & 1) * 8 + (g >> 1) * 16;
  if (P.partial) {  // four fp32 neighbours are 16 bytes as they lie
    float FWDMI_GLOBAL* const out = gmut<float>(P.partial) + (int64_t)split * P.ni * P.nj;
    const int j4 = j0 + wave / WI * (TJ / WJ) + g * 4;
#pragma unroll
    for (int i = 0; i < FI; ++i)
      if (i_lane + i * 16 < P.ni)
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
          Pack<float, 4> v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v.v[e] = acc[j][i][e];
          store_slice<float, 4>(out + (int64_t)(i_lane + i * 16) * P.nj + j4 + j * 16, v);
        }
    return;
  }
  auto eight = [&](int p, int i, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // lane rows of the two blocks: 0 1 2 3 and 4 5 6 7 -> 0 1 4 5 and 2 3 6 7 -> 0 2 4 6 and 1 3 5 7
      auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[2 * p][i][e]), __float_as_uint(acc[2 * p + 1][i][e]),
                                                false, false);
      auto b = __builtin_amdgcn_permlane16_swap(a[0], a[1], false, false);
      v[e] = __uint_as_float(b[0]);
      v[e + 4] = __uint_as_float(b[1]);
    }
  };
  static_assert(sizeof(T) == 2 && FJ == 4, "two slices of 16 bytes per lane and row");
  const bool second = (lane & 8) != 0;
  const int row = i_lane - (lane & 15) + (lane & 7), col = j_lane + (second ? 32 : 0);
  // Slices 0 and 1 of 16 rows, every lane with its row's: lanes eight apart trade one each, so that each store writes whole
  // 128-byte lines of eight rows (half lines cost 8 % more time where the results go to memory).
  auto store_rows = [&](void* to, int i, const Pack<T, 8> (&v)[2]) {
    uint32_t u[2][4];
    __builtin_memcpy(u, v, 32);
    uint32_t low[4], high[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t other0 = __builtin_amdgcn_update_dpp(0, (int)u[0][k], 0x128, 0xf, 0xf, true);  // of the row eight on
      const uint32_t other1 = __builtin_amdgcn_update_dpp(0, (int)u[1][k], 0x128, 0xf, 0xf, true);
      low[k] = second ? other1 : u[0][k];
      high[k] = second ? u[1][k] : other0;
    }
    Pack<T, 8> o;
    T FWDMI_GLOBAL* const at = gmut<T>(to) + (int64_t)(row + i * 16) * P.nj + col;
    if (row + i * 16 < P.ni) {
      __builtin_memcpy(&o, low, 16);
      store_slice<T, 8>(at, o);
    }
    if (row + i * 16 + 8 < P.ni) {
      __builtin_memcpy(&o, high, 16);
      store_slice<T, 8>(at + 8 * (int64_t)P.nj, o);
    }
  };
  with_act(EPILOGUE ? P.act : FWDMI_ACT_NONE, [&](auto act) {
    if (!EPILOGUE && decltype(act)::value != FWDMI_ACT_NONE) return;
    float b[2][8] = {};
    if (EPILOGUE)
#pragma unroll
      for (int p = 0; p < 2; ++p) load_bias(P, j_lane + p * 32, b[p]);
#pragma unroll
    for (int i = 0; i < FI; ++i) {
      const int ii = i_lane + i * 16;
      Pack<T, 8> y[2], z[2], r[2] = {};
      if (EPILOGUE && P.residual && ii < P.ni)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          r[p] = load_slice<T, 8>(gconst<T>(P.residual) + (int64_t)ii * P.nj + j_lane + p * 32);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float v[8];
        eight(p, i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float s = v[e] + b[p][e];
          z[p].v[e] = (T)s;
          y[p].v[e] = (T)(activate<decltype(act)::value, false>(s) + (float)r[p].v[e]);
        }
      }
      store_rows(P.c, i, y);
      if (EPILOGUE && P.preact) store_rows(P.preact, i, z);
    }
  });
}

// The work of workgroup `block` of `blocks` on product P.  Products of these sizes are bound by the latency of their few
// steps and by what a CU loads, 90 KB/us (384 x 1024 x 4096 fp16: 10.5 us, 306 TFLOP/s, of which 7.1 are its 640 KB), or, in fp32, by the matrix
// instructions and LDS in turn (1003 x 517 x 1024: 15.5 us, 69 TFLOP/s; 8192 x 1024 x 4096: 126, where a large library
// product reaches 145).  The waves are WI x WJ over the tile and WK over the halves of
// a step (their sums meet in LDS): small tiles, whose waves would otherwise have little to do between two barriers.
template <typename T, int LA, int LB, int TI, int TJ, int WI, int WJ, int WK, int STEP, int STAGES, bool DIRECT>
struct Work {
  static constexpr int kThreads = 64 * WI * WJ * WK;
  static constexpr int kRoom = STAGES * (TI + TJ) * STEP;  // bytes of LDS
  __device__ static __forceinline__ void run(const Product& P, char* s_tile, int block, int blocks);
};
template <typename T, int LA, int LB, int TI, int TJ, int WI, int WJ, int WK, int STEP, int STAGES, bool DIRECT>
__device__ __forceinline__ void Work<T, LA, LB, TI, TJ, WI, WJ, WK, STEP, STAGES, DIRECT>::run(const Product& P, char* s_tile,
                                                                                               int block, int blocks) {
  constexpr int kNT = 64 * WI * WJ * WK;
  constexpr int kFI = TI / WI / 16, kFJ = TJ / WJ / 16, kHalves = STEP / 64 / WK;
  using TileA = Tile<T, TI, LA, STEP>;
  using TileB = Tile<T, TJ, LB, STEP>;
  using LoadA = Loader<T, TI, LA, STEP, kNT, DIRECT>;
  using LoadB = Loader<T, TJ, LB, STEP, kNT, DIRECT>;
  static_assert(DIRECT || STAGES == 2, "registers hold one step");
  constexpr int kBuffer = TileA::kBytes + TileB::kBytes;  // one step of both operands
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int i0, j0;
  const int split = locate_tile<TI, TJ>(P, block, blocks, i0, j0);
  const int wi = wave % WI * (TI / WI), wj = wave / WI % WJ * (TJ / WJ), wk = wave / (WI * WJ);

  const Steps steps = split_steps(P, split);

  F4 acc[kFJ][kFI];
#pragma unroll
  for (int j = 0; j < kFJ; ++j)
#pragma unroll
    for (int i = 0; i < kFI; ++i) acc[j][i] = F4{0.0f, 0.0f, 0.0f, 0.0f};

  const Reader<T, TI, LA, STEP, kFI> ra(wi);
  const Reader<T, TJ, LB, STEP, kFJ> rb(wj);
  auto multiply_step = [&](const char* now) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      Frag<T> fa[kFI], fb[kFJ];
      ra.read(now, wk * kHalves + h, fa);
      rb.read(now + TileA::kBytes, wk * kHalves + h, fb);
      multiply_all<T>(fb, fa, acc);
    }
  };
  if constexpr (DIRECT) {
    LoadA la(P.a, P.lda, i0, P.ni, steps.first, steps.whole, P.nt - steps.first * TileA::kT);
    LoadB lb(P.b, P.ldb, j0, P.nj, steps.first, steps.whole, P.nt - steps.first * TileB::kT);
    // STAGES - 1 steps of loads are in flight; steps past the end load nothing (every lane out of range) so that the
    // number in flight is always the same
    constexpr int kAhead = (STAGES - 2) * (LoadA::kLoads + LoadB::kLoads);
    static_assert(kAhead < 64, "what the counter of loads in flight holds");
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k) {
      la.load(s_tile + k * kBuffer);
      lb.load(s_tile + k * kBuffer + TileA::kBytes);
    }
    int now = 0, next = (STAGES - 1) * kBuffer;
    if (steps.tail > 0) {
      // The end of t comes first, through the buffer that nothing is on its way to: its loads, which have to be waited for,
      // take the time that the first steps' take anyway.
      la.tail(s_tile + next, steps.whole - (STAGES - 1), steps.tail);
      lb.tail(s_tile + next + TileA::kBytes, steps.whole - (STAGES - 1), steps.tail);
      __syncthreads();
      multiply_step(s_tile + next);
    }
    for (int s = 0; s < steps.whole; ++s) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(wait_loads(kAhead));  // this step's are in
      __builtin_amdgcn_s_barrier();                    // ... of every wave, and the buffer of the step before has been read
      __builtin_amdgcn_sched_barrier(0);
      la.load(s_tile + next);
      lb.load(s_tile + next + TileA::kBytes);
      multiply_step(s_tile + now);
      now = now + kBuffer == STAGES * kBuffer ? 0 : now + kBuffer;
      next = next + kBuffer == STAGES * kBuffer ? 0 : next + kBuffer;
    }
    __builtin_amdgcn_s_waitcnt(wait_loads(0));  // loads past the end write zeros: before the buffers are used again
  } else if (const int n = steps.whole + (steps.tail > 0 ? 1 : 0); n > 0) {
    const int t = steps.whole * TileA::kT + steps.tail;
    LoadA la(P.a, P.lda, i0, P.ni, steps.first, n, t);
    LoadB lb(P.b, P.ldb, j0, P.nj, steps.first, n, t);
    // registers hold the two steps after the one being multiplied
    la.template fetch<0>();
    lb.template fetch<0>();
    la.template drop<0>(s_tile);
    lb.template drop<0>(s_tile + TileA::kBytes);
    la.template fetch<1>();
    lb.template fetch<1>();
    auto step = [&](auto set, int s) {
      constexpr int kSet = decltype(set)::value;  // s & 1
      char* const next = s_tile + (kSet ^ 1) * kBuffer;
      __syncthreads();  // this step's tiles are in LDS, and the other buffers have been read
      la.template fetch<kSet>();
      lb.template fetch<kSet>();
      multiply_step(s_tile + kSet * kBuffer);
      if (s + 1 < n) {
        la.template drop<kSet ^ 1>(next);
        lb.template drop<kSet ^ 1>(next + TileA::kBytes);
      }
    };
    for (int s = 0; s < n; s += 2) {
      step(std::integral_constant<int, 0>{}, s);
      if (s + 1 < n) step(std::integral_constant<int, 1>{}, s + 1);
    }
  }
  leave_tile<T, TI, TJ, WI, WJ, WK, STAGES * kBuffer, LA == kAlong && LB == kAlong>(P, acc, s_tile, i0, j0, split);
}

template <typename W>
__global__ __launch_bounds__(W::kThreads) void product_kernel(const Product P) {
  __shared__ __attribute__((aligned(1024))) char s_tile[W::kRoom];
  W::run(P, s_tile, (int)blockIdx.x, (int)gridDim.x);
}

// Both products of a small gradient and dbias in one launch (771 x 1011 x 768 fp16: 11.6 us, bound by the latency of each
// workgroup's steps; 1.5 us of arithmetic): workgroups of dx, of dw, and of 64 columns of dbias each.
template <typename T, int TILE, bool DIRECT>
__global__ __launch_bounds__(TILE * 8) void gradients_kernel(const Gradients G) {
  using X = Work<T, kAlong, kAcross, TILE, TILE, TILE / 32, 1, 4, 256, 2, DIRECT>;
  using W = Work<T, kAcross, kAcross, TILE, TILE, TILE / 32, 1, 4, 256, 2, DIRECT>;
  static_assert(X::kThreads == TILE * 8 && W::kThreads == X::kThreads && X::kRoom == W::kRoom, "one shape of workgroup");
  __shared__ __attribute__((aligned(1024))) char s_tile[X::kRoom];
  const int b = (int)blockIdx.x;
  if (b < G.blocks_x) {
    X::run(G.x, s_tile, b, G.blocks_x);
  } else if (b < G.blocks_x + G.blocks_w) {
    W::run(G.w, s_tile, b - G.blocks_x, G.blocks_w);
  } else {
    float(*s_red)[64] = reinterpret_cast<float(*)[64]>(s_tile);
    const int64_t c = (int64_t)(b - G.blocks_x - G.blocks_w) * 64 + (threadIdx.x & 63);
    const float a = G.part ? column_sum<float, TILE / 8>(G.part, G.parts, G.n, c, s_red)
                           : column_sum<T, TILE / 8>(static_cast<const T*>(G.dy), G.parts, G.n, c, s_red);
    if (threadIdx.x < 64 && c < G.n) gmut<float>(G.dbias)[c] = a;
  }
}

template <int... I, typename F>
__device__ __forceinline__ void unrolled(std::integer_sequence<int, I...>, F&& f) {
  (f(std::integral_constant<int, I>{}), ...);
}

// Large products of 16-bit operands: eight waves, two on every SIMD of the CU, take turns.  While one multiplies (16
// matrix instructions, 256 cycles of its SIMD), the other reads the fragments of its next 16 from LDS, and both change
// over at a barrier.  Waves 4 .. 7 run half a phase behind 0 .. 3, by one barrier more in front and one fewer behind.
//
// Bound by the matrix cores where the operands are warm (8192 x 4096 x 1024 bf16: 64 us, 1.07 PFLOP/s), by the loads' way
// from memory and the results' way there where they are cold (75 us); an erf GELU and its stored z add 20 us, for 134 MB
// of results leave together.  rocprofv3 counts no LDS bank conflict, and matrix instructions in 0.4 of the busy cycles.
//
// A step of 64 t has a phase for each half of t and each 64 rows of the wave.  With two buffers (256 x 256 tiles, 128 KB)
// the next step's loads go into the buffer of the step before this one: they start in phase 1, when the late waves
// have read that buffer's last fragments (those reads are waited for in front of the multiplications they feed), and every
// wave waits for its own in the last phase, in front of the barrier behind which the first waves read them.  With
// three buffers (256 x 128, 144 KB; 128 x 128, 96 KB) the loads of the step after next go out in phase 1 and have a whole step more.
template <typename T, int LA, int LB, int TI, int TJ, int WI, int WJ, int STEP, int STAGES>
__global__ __launch_bounds__(512) void product_turns_kernel(const Product P) {
  constexpr int kNT = 512;
  constexpr int kFI = TI / WI / 16, kFJ = TJ / WJ / 16, kQ = kFI / 4, kPhases = STEP / 64 * kQ;
  static_assert(WI * WJ == 8 && kFI % 4 == 0 && kPhases >= 2 && (STAGES >= 3 || kPhases == 4),
                "shape of the phases");
  using TileA = Tile<T, TI, LA, STEP>;
  using TileB = Tile<T, TJ, LB, STEP>;
  using LoadA = Loader<T, TI, LA, STEP, kNT, true>;
  using LoadB = Loader<T, TJ, LB, STEP, kNT, true>;
  constexpr int kBuffer = TileA::kBytes + TileB::kBytes;
  constexpr int kAhead = (STAGES - 2) * (LoadA::kLoads + LoadB::kLoads);  // loads that stay in flight over a step's end
  __shared__ __attribute__((aligned(1024))) char s_tile[STAGES * kBuffer];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int i0, j0;
  const int split = locate_tile<TI, TJ>(P, (int)blockIdx.x, (int)gridDim.x, i0, j0);
  const int wi = wave % WI * (TI / WI), wj = wave / WI * (TJ / WJ);
  const Steps steps = split_steps(P, split);

  F4 acc[kFJ][kFI];
#pragma unroll
  for (int j = 0; j < kFJ; ++j)
#pragma unroll
    for (int i = 0; i < kFI; ++i) acc[j][i] = F4{0.0f, 0.0f, 0.0f, 0.0f};

  LoadA la(P.a, P.lda, i0, P.ni, steps.first, steps.whole, P.nt - steps.first * TileA::kT);
  LoadB lb(P.b, P.ldb, j0, P.nj, steps.first, steps.whole, P.nt - steps.first * TileB::kT);
  const Reader<T, TI, LA, STEP, kFI> ra(wi);
  const Reader<T, TJ, LB, STEP, kFJ> rb(wj);
  // (steps past the end load nothing, every lane out of range, so that the number in flight is always the same)
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) {
    la.load(s_tile + k * kBuffer);
    lb.load(s_tile + k * kBuffer + TileA::kBytes);
  }
  Frag<T> fa[4], fb[kFJ];
  auto change = [&] {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply_block = [&](auto first) {
    constexpr int kFirst = decltype(first)::value;
#pragma unroll
    for (int j = 0; j < kFJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][kFirst + i] = multiply<T>(fb[j], fa[i], acc[j][kFirst + i]);
  };
  int now_at = 0, next_at = (STAGES - 1) * kBuffer;
  if (steps.tail > 0) {  // the end of t comes first, as in Work
    char* const end = s_tile + next_at;
    la.tail(end, steps.whole - (STAGES - 1), steps.tail);
    lb.tail(end + TileA::kBytes, steps.whole - (STAGES - 1), steps.tail);
    __syncthreads();
    unrolled(std::make_integer_sequence<int, kPhases>{}, [&](auto phase) {
      constexpr int ph = decltype(phase)::value, h = ph / kQ, q = ph % kQ;
      if constexpr (q == 0) rb.read(end + TileA::kBytes, h, fb);
      ra.template read<q * 4, 4>(end, h, fa);
      multiply_block(std::integral_constant<int, q * 4>{});
    });
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(wait_loads(kAhead));
  __builtin_amdgcn_s_barrier();
  if (wave >= 4) __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  for (int s = 0; s < steps.whole; ++s) {
    const char* const now = s_tile + now_at;
    char* const next = s_tile + next_at;
    unrolled(std::make_integer_sequence<int, kPhases>{}, [&](auto phase) {
      constexpr int ph = decltype(phase)::value, h = ph / kQ, q = ph % kQ;
      if constexpr (q == 0) rb.read(now + TileA::kBytes, h, fb);
      ra.template read<q * 4, 4>(now, h, fa);
      if constexpr (ph == 1) la.load(next);
      if constexpr (ph == (STAGES == 2 ? 2 : 1)) lb.load(next + TileA::kBytes);
      if constexpr (ph == kPhases - 1) __builtin_amdgcn_s_waitcnt(wait_loads(kAhead));
      change();
      __builtin_amdgcn_s_setprio(1);
      multiply_block(std::integral_constant<int, q * 4>{});
      __builtin_amdgcn_s_setprio(0);
      change();
    });
    now_at = now_at + kBuffer == STAGES * kBuffer ? 0 : now_at + kBuffer;
    next_at = next_at + kBuffer == STAGES * kBuffer ? 0 : next_at + kBuffer;
  }
  if (wave < 4) __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_s_waitcnt(wait_loads(0));  // loads past the end write zeros: before the buffers are used again
  if constexpr (kFJ == 4) {  // (a wave's 64 columns are whole 128-byte lines)
    if (j0 + TJ <= P.nj)
      return leave_registers<T, TI, TJ, WI, WJ, LA == kAlong && LB == kAlong>(P, acc, i0, j0, split);
  }
  leave_tile<T, TI, TJ, WI, WJ, 1, STAGES * kBuffer, LA == kAlong && LB == kAlong>(P, acc, s_tile, i0, j0, split);
}

// A few rows (at most 16 MB tokens) through a matrix of weights: one pass over w, which bounds it.  1 x 4096 x 1024 fp16
// (8.4 MB): 4.0 us, of which 2 are a launch's own and the rest one trip to memory per wave.  A workgroup takes 16 rows of w and
// all of x; its waves take 128-byte pieces of t in turn, straight from memory to the matrix instructions (a piece is
// read by one wave alone, LDS would only add a stop), two pieces in flight, and their sums meet in LDS in wave order.
// Rows past the last repeat it, their products are dropped.  blockIdx.y: splits of the pieces (few rows of w, long ones).
template <typename T, int MB>
__global__ __launch_bounds__(1024) void product_few_kernel(const Product P) {
  extern __shared__ __attribute__((aligned(16))) F4 s_sum[];  // [waves][MB][64]
  constexpr int kPiece = 128 / (int)sizeof(T), kHalf = kPiece / 2;
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int j0 = (int)blockIdx.x * 16;
  const T FWDMI_GLOBAL* const pw = gconst<T>(P.b) + (int64_t)min(j0 + r, P.nj - 1) * P.ldb + g * kChunk<T>;
  const T FWDMI_GLOBAL* px[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) px[b] = gconst<T>(P.a) + (int64_t)min(b * 16 + r, P.ni - 1) * P.lda + g * kChunk<T>;
  F4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = F4{0.0f, 0.0f, 0.0f, 0.0f};

  const int split = (int)blockIdx.y, pieces = min(P.nt / kPiece, (split + 1) * P.steps_per_split);
  constexpr int kBatch = 2;
  auto batch = [&](int piece, auto count) {
    constexpr int kN = decltype(count)::value;
    Frag<T> w[kN][2], x[kN][2][MB];
#pragma unroll
    for (int k = 0; k < kN; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t t = (int64_t)(piece + k * waves) * kPiece + h * kHalf;
        w[k][h].v = load_slice<T, kChunk<T>>(pw + t);
#pragma unroll
        for (int b = 0; b < MB; ++b) x[k][h][b].v = load_slice<T, kChunk<T>>(px[b] + t);
      }
#pragma unroll
    for (int k = 0; k < kN; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[b] = multiply<T>(w[k][h], x[k][h][b], acc[b]);
  };
  int piece = split * P.steps_per_split + wave;
  for (; piece + (kBatch - 1) * waves < pieces; piece += kBatch * waves) batch(piece, std::integral_constant<int, kBatch>{});
  for (; piece < pieces; piece += waves) batch(piece, std::integral_constant<int, 1>{});
  // the wave whose turn it is in the last split takes what is left, element by element
  if (piece == pieces && split + 1 == (int)gridDim.y && P.nt % kPiece != 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = pieces * kPiece + h * kHalf, n = P.nt - t - g * kChunk<T>;
      auto some = [&](const T FWDMI_GLOBAL* p) {
        Frag<T> f;
#pragma unroll
        for (int e = 0; e < kChunk<T>; ++e) f.v.v[e] = e < n ? p[t + e] : (T)0.0f;
        return f;
      };
      const Frag<T> w = some(pw);
#pragma unroll
      for (int b = 0; b < MB; ++b) acc[b] = multiply<T>(w, some(px[b]), acc[b]);
    }
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) s_sum[(wave * MB + b) * 64 + lane] = acc[b];
  __syncthreads();
  if (wave < MB) {
    float v[4] = {};
    for (int k = 0; k < waves; ++k) {
      const F4 part = s_sum[(k * MB + wave) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += part[e];
    }
    const int i = wave * 16 + r, j = j0 + g * 4;
    if (P.partial && i < P.ni) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < P.nj) gmut<float>(P.partial)[((int64_t)split * P.ni + i) * P.nj + j + e] = v[e];
    } else if (i < P.ni && j < P.nj) {
      float b[4];
      load_bias(P, j, b);
      with_act(P.act, [&](auto act) { finish<T, decltype(act)::value>(P, i, j, v, b); });
    }
  }
}

// Adds the splits' partial products in split order and finishes them; bound by memory (four splits of 4096 x 1024: 75 MB in
// 13 us, 5.8 TB/s, the partials partly from cache); eight neighbours of a row per lane.
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(const Product P, int splits) {
  const uint32_t per = (P.nj + 7) / 8;
  const uint32_t q = blockIdx.x * 256 + threadIdx.x;  // (a launch holds fewer than 2^32 lanes)
  const int64_t i = q / per;
  if (i >= P.ni) return;
  const int j = (int)(q % per) * 8;
  const int64_t plane = (int64_t)P.ni * P.nj;
  const float FWDMI_GLOBAL* p = gconst<float>(P.partial) + i * P.nj + j;
  const int live = min(P.nj - j, 8);
  float acc[8] = {};
  if (live == 8) {
    constexpr int kBatch = 4;  // splits in flight
    for (int s = 0; s < splits; s += kBatch) {
      Pack<float, 4> lo[kBatch], hi[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float FWDMI_GLOBAL* const q = p + min(s + k, splits - 1) * plane;
        lo[k] = load_slice<float, 4>(q);
        hi[k] = load_slice<float, 4>(q + 4);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (s + k < splits)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[e] += lo[k].v[e];
            acc[e + 4] += hi[k].v[e];
          }
    }
  } else {
    for (int s = 0; s < splits; ++s, p += plane)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < live) acc[e] += p[e];
  }
  float b[8];
  load_bias(P, j, b);
  with_act(P.act, [&](auto act) { finish<T, decltype(act)::value>(P, i, j, acc, b); });
}

// ---- dz = dy * act'(z) and its column sums -----------------------------------------------------------------------

// Bound by memory: 8192 x 4096 bf16, 201 MB, 46 us (4.4 TB/s; a large copy reaches 5.2).  512 columns (8 per lane) x every (4 gridDim.y)-th row per wave, the four waves' sums through LDS.
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
        T FWDMI_GLOBAL* const to = gmut<T>(S.dz) + r * S.ld_dz + c;
        if (c + kVec <= S.ld_dz) {  // (elements past n come out as zeros)
          store_slice<T, kVec>(to, out);
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (e < live) to[e] = out.v[e];
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

template <typename T>
int launch_finish(const Product& P, int splits, hipStream_t stream) {
  const int64_t octets = (int64_t)P.ni * ((P.nj + 7) / 8);
  if (const int rc = check_launch((octets + 255) / 256, 256)) return rc;
  hipLaunchKernelGGL((finish_kernel<T>), dim3((unsigned)ceil_div(octets, 256)), dim3(256), 0, stream, P, splits);
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

template <typename T, int LA, int LB, bool DIRECT>
int launch_product(Product& P, const Plan& plan, hipStream_t stream) {
  if constexpr (LA == kAlong && LB == kAlong) {
    if (plan.tile == kFew) {
      const int pieces = plan.steps_per_split;
      const int waves = pieces >= 32 ? 16 : pieces >= 16 ? 8 : 4;
      P.steps_per_split = pieces;
      const dim3 grid((unsigned)ceil_div(P.nj, 16), (unsigned)plan.splits), block(64 * waves);
      if (const int rc = check_launch((int64_t)grid.x * grid.y, 64 * waves)) return rc;
      if (P.ni <= 16)
        hipLaunchKernelGGL((product_few_kernel<T, 1>), grid, block, waves * 1024, stream, P);
      else
        hipLaunchKernelGGL((product_few_kernel<T, 2>), grid, block, waves * 2048, stream, P);
      FWDMI_HIP_CHECK(hipGetLastError());
      return plan.splits > 1 ? launch_finish<T>(P, plan.splits, stream) : FWDMI_OK;
    }
  }
  const TileShape tile = kTiles[plan.tile];
  P.tiles_i = ceil_div(P.ni, tile.ti);
  P.tiles_j = ceil_div(P.nj, tile.tj);
  P.whole_steps = plan.whole_steps;
  P.tail = plan.tail;
  P.steps_per_split = plan.steps_per_split;
  const int64_t tiles = (int64_t)P.tiles_i * P.tiles_j * plan.splits;
  if (const int rc = check_launch(tiles, 512)) return rc;
  const dim3 grid((unsigned)tiles);
#define FWDMI_PRODUCT(KIND_, ...)                                                                                  \
  if (plan.tile == KIND_) {                                                                                       \
    using W = Work<T, LA, LB, __VA_ARGS__, DIRECT>;                                                               \
    hipLaunchKernelGGL((product_kernel<W>), grid, dim3(W::kThreads), 0, stream, P);                               \
  }
  constexpr bool kHalf = sizeof(T) == 2, kBothAlong = LA == kAlong && LB == kAlong;
  if constexpr (kHalf && DIRECT) {
    if (plan.tile == k256x256)
      hipLaunchKernelGGL((product_turns_kernel<T, LA, LB, 256, 256, 2, 4, 128, 2>), grid, dim3(512), 0, stream, P);
    if (plan.tile == k256x128)
      hipLaunchKernelGGL((product_turns_kernel<T, LA, LB, 256, 128, 4, 2, 128, 3>), grid, dim3(512), 0, stream, P);
    if (plan.tile == k128x128Turns)
      hipLaunchKernelGGL((product_turns_kernel<T, LA, LB, 128, 128, 2, 4, 128, 3>), grid, dim3(512), 0, stream, P);
  }
  FWDMI_PRODUCT(k128x128, 128, 128, 2, 2, 1, 128, 2)
  FWDMI_PRODUCT(k64x64, 64, 64, 2, 1, 4, 256, 2)
  if constexpr (DIRECT) {
    FWDMI_PRODUCT(k32x32Deep, 32, 32, 1, 1, 8, 512, 3)
    if constexpr (kHalf && kBothAlong) {
      FWDMI_PRODUCT(k64x64Alone, 64, 64, 2, 1, 4, 256, 3)
      FWDMI_PRODUCT(k48x32, 48, 32, 1, 1, 8, 512, 3)
    } else {
      FWDMI_PRODUCT(k64x64Alone, 64, 64, 1, 1, 8, 512, 2)
    }
  }
  if constexpr (kHalf && DIRECT) {
    FWDMI_PRODUCT(k64x32, 64, 32, 2, 1, 4, 512, 3)
  } else {
    FWDMI_PRODUCT(k64x32, 64, 32, 2, 1, 4, 256, (DIRECT ? 4 : 2))
  }
  if constexpr (!kHalf) {
    FWDMI_PRODUCT(k32x32, 32, 32, 1, 1, 4, 256, 2)
    if constexpr (DIRECT && kBothAlong) {
      FWDMI_PRODUCT(k48x48, 48, 48, 1, 1, 8, 512, 3)
    }
  }
#undef FWDMI_PRODUCT
  FWDMI_HIP_CHECK(hipGetLastError());
  return plan.splits > 1 ? launch_finish<T>(P, plan.splits, stream) : FWDMI_OK;
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
int run_gradients(const Gradients& G, bool direct, hipStream_t stream) {
  const int64_t blocks = (int64_t)G.blocks_x + G.blocks_w + (G.dbias ? ceil_div(G.n, 64) : 0);
  if (const int rc = check_launch(blocks, kTiles[G.tile].ti * 8)) return rc;
  const dim3 grid((unsigned)blocks);
  if (G.tile == k64x64) {
    if (direct)
      hipLaunchKernelGGL((gradients_kernel<T, 64, true>), grid, dim3(512), 0, stream, G);
    else
      hipLaunchKernelGGL((gradients_kernel<T, 64, false>), grid, dim3(512), 0, stream, G);
  }
  if constexpr (sizeof(T) == 4) {
    if (G.tile == k32x32) {
      if (direct)
        hipLaunchKernelGGL((gradients_kernel<T, 32, true>), grid, dim3(256), 0, stream, G);
      else
        hipLaunchKernelGGL((gradients_kernel<T, 32, false>), grid, dim3(256), 0, stream, G);
    }
  }
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}
template <typename T>
int run_slope(const Slope& S, int parts, hipStream_t stream) {
  const dim3 grid((unsigned)ceil_div(S.n, 512), (unsigned)parts);
  if (const int rc = check_launch((int64_t)grid.x * grid.y, 256)) return rc;
  hipLaunchKernelGGL((slope_kernel<T>), grid, dim3(256), 0, stream, S);
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

}  // namespace
}  // namespace fwdmi
