// LayerNorm for training on gfx950: the forward pass that keeps its statistics (and, for pre-norm layers, the
// sum it normalises) and the backward pass with the column sums of gamma's, beta's and the bias's gradients.
//
//   h = x (+ skip) (+ bias),  mean and rstd = 1 / sqrt(var + eps) over a row,  xhat = (h - mean) * rstd
//   y = gamma * xhat + beta
//   dh = rstd * (g - mean(g) - xhat * mean(g * xhat)) with g = dy * gamma,  dx = dh (+ dsum)
//   dgamma = sum over rows of dy * xhat, dbeta = sum of dy, dbias = sum of dx
//
// Everything between the loads and the one rounding at the store is fp32.  LPR lanes own a row (a part of a
// wavefront, a wavefront, or several), 16 bytes per lane and step, NV steps, the row in registers: it is read
// once, and the next row's loads are in flight while this one is reduced.  Rows that do not divide into 16-byte
// slices (odd lengths, any element alignment) use the same loads unaligned: the lane that holds the row's end
// reads the row's LAST slice instead and leaves out the elements its neighbour has.
//
// The column sums stay in registers over all rows a workgroup processes, are combined through LDS in a fixed
// order and leave as one row of partials per workgroup; a second small launch adds those, also in a fixed order:
// no atomics, results repeat bit for bit.  Longer rows have their column sums computed by a kernel that walks down the
// rows (ln_backward_columns_kernel), and rows longer than a workgroup's registers are streamed from cache
// (ln_*_stream_kernel).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "slice.h"

// No implicit multiply-add fusion: every variant of a kernel (with a bias, from a stored sum, any lane layout) rounds
// the same operations the same way, so every fused operation is written as an explicit fma.
#pragma clang fp contract(off)

namespace fwdmi {
namespace {

struct LnTrain {
  const void* x;
  const void* skip;  // nullable
  const void* dsum;  // backward, nullable: gradient that arrives at the sum from elsewhere
  const void* dy;    // backward
  const float* gamma;
  const float* beta;  // forward
  const float* bias;  // nullable
  void* out;          // forward: y; backward: dx
  void* sum;          // forward, nullable: h rounded to T
  float* mean;        // forward: written; backward: read
  float* rstd;
  float* part_gamma;  // backward: row p of partials starts at part_* + p * part_stride
  float* part_beta;
  float* part_bias;
  float* c1;          // backward of long rows: mean(g * xhat) and mean(g) per row
  float* c2;
  int64_t part_stride;
  int64_t rows;
  int32_t ld;
  int32_t row_blocks;  // backward: workgroups of rows; those behind them sum columns (see ln_columns)
  float eps;
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Sum over aligned groups of G lanes (G = 8 .. 64), the same value in every lane of the group.
template <int G>
__device__ __forceinline__ float group_sum(float x) {
  x = dpp_add<0xB1>(x);              // lane ^ 1
  x = dpp_add<0x4E>(x);              // lane ^ 2
  x = dpp_add<0x141>(x);             // the other quad of each 8
  if (G >= 16) x = dpp_add<0x140>(x);  // the other half of each row of 16
  if (G >= 32) x += __shfl_xor(x, 16);
  if (G >= 64) x += __shfl_xor(x, 32);
  return x;
}

// Sum over the LPR lanes of a row; `scratch` holds WG / 64 floats per use and phase of the caller's loop.
template <int WG, int LPR>
__device__ __forceinline__ float row_sum(float x, float* scratch) {
  if constexpr (LPR <= 64) {
    return group_sum<LPR>(x);
  } else {
    constexpr int kWaves = LPR / 64;
    const int wave = threadIdx.x >> 6;
    x = group_sum<64>(x);
    if ((threadIdx.x & 63) == 0) scratch[wave] = x;
    __syncthreads();
    const int first = wave / kWaves * kWaves;
    float s = scratch[first];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) s += scratch[first + k];
    return s;
  }
}

// 1 / sqrt(v) to 1 ulp.  The instruction takes subnormal numbers for zero: rows of values near 1e-19 (fp32, bf16) without an
// eps have such variances, and are scaled by powers of two, which changes no bit of any other row's result.
__device__ __forceinline__ float inverse_root(float v) {
  const bool small = v < 0x1p-100f;
  return __builtin_amdgcn_rsqf(small ? v * 0x1p100f : v) * (small ? 0x1p50f : 1.0f);
}

// Where a lane's slices lie: columns col[j] .. col[j] + VEC, of which the first drop[j] belong to another lane
// (the row's end) or to nobody (drop == VEC).  FULL: ld == LPR * VEC * NV, every element is the lane's own.
template <int VEC, int NV, int LPR, bool FULL>
struct Columns {
  int col[NV];
  int drop[NV];
  __device__ __forceinline__ Columns(int lane_in_row, int ld) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane_in_row) * VEC;
      if (FULL || c + VEC <= ld) {
        col[j] = c;
        drop[j] = 0;
      } else if (c < ld) {
        col[j] = ld - VEC;
        drop[j] = VEC - (ld - c);
      } else {
        col[j] = 0;
        drop[j] = VEC;
      }
    }
  }
  __device__ __forceinline__ bool own(int j, int e) const { return FULL || e >= drop[j]; }
  // Stores the lane's own elements of slice j (the row's end one by one, at most one lane of the row).
  template <typename T>
  __device__ __forceinline__ void store(T FWDMI_GLOBAL* row, int j, const Pack<T, VEC>& o) const {
    if (FULL || drop[j] == 0) {
      store_slice<T, VEC>(row + col[j], o);
    } else if (VEC > 1 && drop[j] < VEC) {
#pragma unroll
      for (int e = 1; e < VEC; ++e)
        if (e >= drop[j]) row[col[j] + e] = o.v[e];
    }
  }
};

// Bound by memory: every operand passes once.  8192 x 1024 fp16 with a skip moves its 50 MB in 10.1 us (5.0 TB/s; a large
// copy reaches 5.2), 8192 x 4096 bf16 with a skip and a stored sum its 268 MB in 41 us (part of it from cache; 52 us where
// all comes from memory), one row of 1024 takes 2.3 us, a launch's own time.  Variance from the differences to the mean
// (a second sum over registers): no cancellation, and it costs nothing next to the loads.
template <typename T, int VEC, int NV, int WG, int LPR, bool FULL>
__global__ __launch_bounds__(WG) void ln_forward_kernel(const LnTrain L) {
  constexpr int kRows = WG / LPR;
  __shared__ float s_red[4 * (WG / 64)];
  const int gl = threadIdx.x % LPR;
  const int group = threadIdx.x / LPR;
  const Columns<VEC, NV, LPR, FULL> C(gl, L.ld);
  const T FWDMI_GLOBAL* const px = gconst<T>(L.x);
  const T FWDMI_GLOBAL* const ps = gconst<T>(L.skip);
  const bool has_skip = L.skip != nullptr;

  Pack<T, VEC> x[NV], s[NV];
  auto fetch = [&](int64_t r) {
    const int64_t base = min(r, L.rows - 1) * L.ld;  // groups past the last row repeat it and store nothing
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j] = load_slice<T, VEC>(px + base + C.col[j]);
      if (has_skip) s[j] = load_slice<T, VEC>(ps + base + C.col[j]);
    }
  };

  const int64_t step = (int64_t)gridDim.x * kRows;
  const int64_t first = (int64_t)blockIdx.x * kRows;
  fetch(first + group);
  float g[NV][VEC], be[NV][VEC], bi[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Pack<float, VEC> pg = load_slice<float, VEC>(gconst<float>(L.gamma) + C.col[j]);
    const Pack<float, VEC> pb = load_slice<float, VEC>(gconst<float>(L.beta) + C.col[j]);
    Pack<float, VEC> pi{};
    if (L.bias) pi = load_slice<float, VEC>(gconst<float>(L.bias) + C.col[j]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      g[j][e] = pg.v[e];
      be[j][e] = pb.v[e];
      bi[j][e] = pi.v[e];
    }
  }
  const float inv_n = 1.0f / (float)L.ld;
  int phase = 0;
  for (int64_t r0 = first; r0 < L.rows; r0 += step, phase ^= 1) {  // the same count for every wave of the workgroup
    const int64_t r = r0 + group;
    const bool row_ok = r < L.rows;
    float h[NV][VEC], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float v = (float)x[j].v[e];
        if (has_skip) v += (float)s[j].v[e];
        v += bi[j][e];
        h[j][e] = v;
        sum += C.own(j, e) ? v : 0.0f;
      }
    if (r0 + step < L.rows) fetch(r + step);
    const float mu = row_sum<WG, LPR>(sum, s_red + phase * 2 * (WG / 64)) * inv_n;
    float m2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = C.own(j, e) ? h[j][e] - mu : 0.0f;
        m2 = __builtin_fmaf(d, d, m2);
      }
    m2 = row_sum<WG, LPR>(m2, s_red + (phase * 2 + 1) * (WG / 64));
    const float rs = inverse_root(__builtin_fmaf(m2, inv_n, L.eps));
    if (row_ok) {
      if (gl == 0) {
        gmut<float>(L.mean)[r] = mu;
        gmut<float>(L.rstd)[r] = rs;
      }
      T FWDMI_GLOBAL* const py = gmut<T>(L.out) + r * L.ld;
      T FWDMI_GLOBAL* const ph = gmut<T>(L.sum) + r * L.ld;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Pack<T, VEC> o;
        if (L.sum) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) o.v[e] = (T)h[j][e];
          C.store(ph, j, o);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = (T)__builtin_fmaf(g[j][e], (h[j][e] - mu) * rs, be[j][e]);
        C.store(py, j, o);
      }
    }
  }
}

// gamma's and beta's gradients of 64 columns straight from dy and x, whose mean and rstd are known: for few rows, whose
// column sums then need no partials and no second launch.  A lane takes 16 bytes of a row, the lanes of a wave several
// rows; their sums are added across the lanes of a column, then across the waves, in a fixed order.
template <typename T, int WG>
__device__ __forceinline__ void ln_columns(const LnTrain& L, int block, float (*s_sum)[2][64]) {
  constexpr int kVec = 16 / sizeof(T), kLanes = 64 / kVec, kWaveRows = 64 / kLanes, kRows = WG / 64 * kWaveRows;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)block * 64 + lane % kLanes * kVec;
  const int live = (int)min((int64_t)kVec, max((int64_t)L.ld - c, (int64_t)0));
  float sg[kVec] = {}, sb[kVec] = {};
  auto some = [&](const void* p, int64_t at) {
    Pack<T, kVec> v{};
    if (live == kVec) {
      v = load_slice<T, kVec>(gconst<T>(p) + at);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e < live) v.v[e] = gconst<T>(p)[at + e];
    }
    return v;
  };
  if (live > 0) {
#pragma unroll 4
    for (int64_t r = wave * kWaveRows + lane / kLanes; r < L.rows; r += kRows) {
      const int64_t at = r * L.ld + c;
      const float mu = gconst<float>(L.mean)[r], rs = gconst<float>(L.rstd)[r];
      const Pack<T, kVec> dy = some(L.dy, at), x = some(L.x, at);
      Pack<T, kVec> s{};
      if (L.skip) s = some(L.skip, at);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        float h = (float)x.v[e];
        if (L.skip) h += (float)s.v[e];
        const float w = (float)dy.v[e];
        sg[e] = __builtin_fmaf(w, (h - mu) * rs, sg[e]);
        sb[e] += w;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
#pragma unroll
    for (int m = kLanes; m < 64; m <<= 1) {
      sg[e] += __shfl_xor(sg[e], m);
      sb[e] += __shfl_xor(sb[e], m);
    }
    if (lane < kLanes) {
      s_sum[wave][0][lane * kVec + e] = sg[e];
      s_sum[wave][1][lane * kVec + e] = sb[e];
    }
  }
  __syncthreads();
  const int kind = (int)threadIdx.x >> 6, col = (int)threadIdx.x & 63;
  if (kind < 2 && (int64_t)block * 64 + col < L.ld) {
    float a = s_sum[0][kind][col];
#pragma unroll
    for (int k = 1; k < WG / 64; ++k) a += s_sum[k][kind][col];
    gmut<float>(kind == 0 ? L.part_gamma : L.part_beta)[(int64_t)block * 64 + col] = a;
  }
}

// Bound by memory and, with the column sums, by the registers that two operands, their successors and three sums per
// element take (one workgroup of 512 or 1024 lanes per CU): 8192 x 1024 bf16 with a skip and a bias, 67 MB, 15.8 us and 3.9 for the sum of
// the partials; 4099 x 1531 fp16 with dsum (no 16-byte alignment), 50 MB, 14.7 and 3.9 us; 509 x 768 fp32 jointly with
// its columns 6.2 us.
//
// SUMS: the column sums ride along in registers.  Rows of more than 16 elements per lane have none left for them
// (2700 x 12288 fp16 took 164 us with the sums spilled): those leave c1 and c2 and ln_backward_columns_kernel reads dy and
// x once more.  Without sums and without a bias the launch may hold workgroups that sum columns (ln_columns).
template <typename T, int VEC, int NV, int WG, int LPR, bool FULL, bool BIAS, bool SUMS>
__global__ __launch_bounds__(WG) void ln_backward_kernel(const LnTrain L) {
  constexpr int kRows = WG / LPR;
  constexpr int kSlots = LPR * NV * VEC;  // elements of a row, as the lanes hold them
  __shared__ float s_red[4 * (WG / 64)];
  __shared__ float s_col[LPR < WG && SUMS ? kRows * kSlots : 1];
  if constexpr (!SUMS && !BIAS) {
    if ((int)blockIdx.x >= L.row_blocks) {
      __shared__ float s_sum[WG / 64][2][64];
      ln_columns<T, WG>(L, (int)blockIdx.x - L.row_blocks, s_sum);
      return;
    }
  }
  const int gl = threadIdx.x % LPR;
  const int group = threadIdx.x / LPR;
  const Columns<VEC, NV, LPR, FULL> C(gl, L.ld);
  const T FWDMI_GLOBAL* const pdy = gconst<T>(L.dy);
  const T FWDMI_GLOBAL* const px = gconst<T>(L.x);
  const T FWDMI_GLOBAL* const ps = gconst<T>(L.skip);
  const T FWDMI_GLOBAL* const pd = gconst<T>(L.dsum);
  const bool has_skip = L.skip != nullptr, has_dsum = L.dsum != nullptr;

  Pack<T, VEC> dy[NV], x[NV], s[NV], d[NV];
  float mu, rs;
  auto fetch = [&](int64_t r) {
    r = min(r, L.rows - 1);
    const int64_t base = r * L.ld;
    mu = gconst<float>(L.mean)[r];
    rs = gconst<float>(L.rstd)[r];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      dy[j] = load_slice<T, VEC>(pdy + base + C.col[j]);
      x[j] = load_slice<T, VEC>(px + base + C.col[j]);
      if (has_skip) s[j] = load_slice<T, VEC>(ps + base + C.col[j]);
      if (has_dsum) d[j] = load_slice<T, VEC>(pd + base + C.col[j]);
    }
  };

  const int64_t step = (int64_t)L.row_blocks * kRows;
  const int64_t first = (int64_t)blockIdx.x * kRows;
  fetch(first + group);
  float g[NV][VEC], bi[NV][VEC], sum_g[NV][VEC], sum_b[NV][VEC], sum_h[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Pack<float, VEC> pg = load_slice<float, VEC>(gconst<float>(L.gamma) + C.col[j]);
    Pack<float, VEC> pi{};
    if (BIAS) pi = load_slice<float, VEC>(gconst<float>(L.bias) + C.col[j]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      g[j][e] = pg.v[e];
      bi[j][e] = pi.v[e];
      sum_g[j][e] = sum_b[j][e] = sum_h[j][e] = 0.0f;
    }
  }
  const float inv_n = 1.0f / (float)L.ld;
  int phase = 0;
  for (int64_t r0 = first; r0 < L.rows; r0 += step, phase ^= 1) {
    const int64_t r = r0 + group;
    const bool row_ok = r < L.rows;
    const float rstd = rs;
    float xh[NV][VEC], gy[NV][VEC], add[NV][VEC], a1 = 0.0f, a2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float h = (float)x[j].v[e];
        if (has_skip) h += (float)s[j].v[e];
        if (BIAS) h += bi[j][e];
        const bool live = row_ok && C.own(j, e);
        const float w = live ? (float)dy[j].v[e] : 0.0f;
        xh[j][e] = (h - mu) * rstd;
        gy[j][e] = w * g[j][e];
        const float xl = live ? xh[j][e] : 0.0f;  // (a column or row of another lane may hold anything)
        a1 = __builtin_fmaf(gy[j][e], xl, a1);
        a2 += gy[j][e];
        if (SUMS) {
          sum_g[j][e] = __builtin_fmaf(w, xl, sum_g[j][e]);
          sum_b[j][e] += w;
        }
        add[j][e] = has_dsum ? (float)d[j].v[e] : 0.0f;
      }
    if (r0 + step < L.rows) fetch(r + step);
    float* const red = s_red + phase * 2 * (WG / 64);
    if constexpr (LPR <= 64) {
      a1 = group_sum<LPR>(a1);
      a2 = group_sum<LPR>(a2);
    } else {  // both sums behind one barrier
      constexpr int kWaves = LPR / 64;
      const int wave = threadIdx.x >> 6;
      a1 = group_sum<64>(a1);
      a2 = group_sum<64>(a2);
      if ((threadIdx.x & 63) == 0) {
        red[wave * 2] = a1;
        red[wave * 2 + 1] = a2;
      }
      __syncthreads();
      const int w0 = wave / kWaves * kWaves;
      a1 = red[w0 * 2];
      a2 = red[w0 * 2 + 1];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) {
        a1 += red[(w0 + k) * 2];
        a2 += red[(w0 + k) * 2 + 1];
      }
    }
    const float c1 = a1 * inv_n, c2 = a2 * inv_n;
    if (!SUMS && L.c1 && row_ok && gl == 0) {
      gmut<float>(L.c1)[r] = c1;
      gmut<float>(L.c2)[r] = c2;
    }
    T FWDMI_GLOBAL* const po = gmut<T>(L.out) + r * L.ld;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float dh = rstd * __builtin_fmaf(-xh[j][e], c1, gy[j][e] - c2);
        const float total = dh + add[j][e];
        if (BIAS && SUMS) sum_h[j][e] += row_ok && C.own(j, e) ? total : 0.0f;
        o.v[e] = (T)total;
      }
      if (row_ok) C.store(po, j, o);
    }
  }

  if constexpr (!SUMS) return;
  // One row of partials per workgroup: the groups' sums in group order.
  auto leave = [&](float (&v)[NV][VEC], float* part) {
    if constexpr (LPR < WG && SUMS) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_col[group * kSlots + (j * LPR + gl) * VEC + e] = v[j][e];
      __syncthreads();
      for (int i = threadIdx.x; i < kSlots; i += WG) {
        float t = s_col[i];
#pragma unroll
        for (int k = 1; k < kRows; ++k) t += s_col[k * kSlots + i];
        // the slice's first column, and the row's last slice where it would pass the row's end
        const int c0 = i / VEC * VEC, e = i % VEC;
        if (FULL || c0 + VEC <= L.ld)
          part[i] = t;
        else if (c0 < L.ld && e >= VEC - (L.ld - c0))
          part[L.ld - VEC + e] = t;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (C.own(j, e)) part[C.col[j] + e] = v[j][e];
    }
  };
  const int64_t p = blockIdx.x * L.part_stride;
  leave(sum_g, L.part_gamma + p);
  leave(sum_b, L.part_beta + p);
  if (BIAS) leave(sum_h, L.part_bias + p);
}

// ---- rows longer than a workgroup's registers ---------------------------------------------------------------

constexpr int kStreamWG = 512;

template <int WG>
__device__ __forceinline__ float wg_sum(float x, float* scratch) {
  __syncthreads();  // the scratch of the sum before this one has been read
  return row_sum<WG, WG>(x, scratch);
}

// Calls f(column, number of elements that exist) for the slices of a row that this lane takes: all of them whole but for
// the row's last, which is a call of its own so that the others compile to vector accesses.
template <int VEC, typename F>
__device__ __forceinline__ void row_slices(int ld, F&& f) {
  int c = (int)threadIdx.x * VEC;
  for (; c + VEC <= ld; c += kStreamWG * VEC) f(c, std::integral_constant<bool, true>{}, VEC);
  if (c < ld) f(c, std::integral_constant<bool, false>{}, ld - c);
}
template <typename T, int VEC, bool WHOLE>
__device__ __forceinline__ void slice_in(const T* p, int64_t at, int n, float (&v)[VEC]) {
  if (WHOLE) {
    const Pack<T, VEC> x = load_slice<T, VEC>(gconst<T>(p) + at);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)x.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = e < n ? (float)gconst<T>(p)[at + e] : 0.0f;
  }
}
template <typename T, int VEC, bool WHOLE>
__device__ __forceinline__ void slice_out(void* p, int64_t at, int n, const float (&v)[VEC]) {
  Pack<T, VEC> o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) o.v[e] = (T)v[e];
  if (WHOLE) {
    store_slice<T, VEC>(gmut<T>(p) + at, o);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e < n) gmut<T>(p)[at + e] = o.v[e];
  }
}
// h of a slice
template <typename T, int VEC, bool WHOLE>
__device__ __forceinline__ void ln_input(const LnTrain& L, int64_t base, int c, int n, float (&h)[VEC]) {
  slice_in<T, VEC, WHOLE>(static_cast<const T*>(L.x), base + c, n, h);
  if (L.skip) {
    float v[VEC];
    slice_in<T, VEC, WHOLE>(static_cast<const T*>(L.skip), base + c, n, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] += v[e];
  }
  if (L.bias) {
    float v[VEC];
    slice_in<float, VEC, WHOLE>(L.bias, c, n, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] += v[e];
  }
}

// A workgroup per row, three passes over it: the first from memory, the others from cache.  2700 x 12288 fp32 (265 MB to
// and from memory): 74 us.
template <typename T>
__global__ __launch_bounds__(kStreamWG) void ln_forward_stream_kernel(const LnTrain L) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float s_red[kStreamWG / 64];
  const float inv_n = 1.0f / (float)L.ld;
  for (int64_t r = blockIdx.x; r < L.rows; r += gridDim.x) {
    const int64_t base = r * L.ld;
    float a = 0.0f;
    row_slices<VEC>(L.ld, [&](int c, auto whole, int n) {
      float h[VEC];
      ln_input<T, VEC, decltype(whole)::value>(L, base, c, n, h);
#pragma unroll
      for (int e = 0; e < VEC; ++e) a += e < n ? h[e] : 0.0f;
    });
    const float mu = wg_sum<kStreamWG>(a, s_red) * inv_n;
    a = 0.0f;
    row_slices<VEC>(L.ld, [&](int c, auto whole, int n) {
      float h[VEC];
      ln_input<T, VEC, decltype(whole)::value>(L, base, c, n, h);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = e < n ? h[e] - mu : 0.0f;
        a = __builtin_fmaf(d, d, a);
      }
    });
    const float rs = inverse_root(__builtin_fmaf(wg_sum<kStreamWG>(a, s_red), inv_n, L.eps));
    if (threadIdx.x == 0) {
      gmut<float>(L.mean)[r] = mu;
      gmut<float>(L.rstd)[r] = rs;
    }
    row_slices<VEC>(L.ld, [&](int c, auto whole, int n) {
      constexpr bool kWhole = decltype(whole)::value;
      float h[VEC], g[VEC], b[VEC];
      ln_input<T, VEC, kWhole>(L, base, c, n, h);
      slice_in<float, VEC, kWhole>(L.gamma, c, n, g);
      slice_in<float, VEC, kWhole>(L.beta, c, n, b);
      if (L.sum) slice_out<T, VEC, kWhole>(L.sum, base + c, n, h);
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[e] = __builtin_fmaf(g[e], (h[e] - mu) * rs, b[e]);
      slice_out<T, VEC, kWhole>(L.out, base + c, n, h);
    });
  }
}

// Two passes, likewise, and the columns' kernel reads dy and x a third time: 2700 x 12288 fp32 takes 146 us in all.  Its three
// planes alone (398 MB) take 77 at a large copy's rate, with dy and x read twice from memory 129.
template <typename T>
__global__ __launch_bounds__(kStreamWG) void ln_backward_stream_kernel(const LnTrain L) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float s_red[kStreamWG / 64];
  const float inv_n = 1.0f / (float)L.ld;
  for (int64_t r = blockIdx.x; r < L.rows; r += gridDim.x) {
    const int64_t base = r * L.ld;
    const float mu = gconst<float>(L.mean)[r], rs = gconst<float>(L.rstd)[r];
    float a1 = 0.0f, a2 = 0.0f;
    row_slices<VEC>(L.ld, [&](int c, auto whole, int n) {
      constexpr bool kWhole = decltype(whole)::value;
      float h[VEC], dy[VEC], g[VEC];
      ln_input<T, VEC, kWhole>(L, base, c, n, h);
      slice_in<T, VEC, kWhole>(static_cast<const T*>(L.dy), base + c, n, dy);
      slice_in<float, VEC, kWhole>(L.gamma, c, n, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float gy = dy[e] * g[e];  // (zeros past the row's end)
        a1 = __builtin_fmaf(gy, (h[e] - mu) * rs, a1);
        a2 += gy;
      }
    });
    const float c1 = wg_sum<kStreamWG>(a1, s_red) * inv_n;
    const float c2 = wg_sum<kStreamWG>(a2, s_red) * inv_n;
    if (threadIdx.x == 0) {
      gmut<float>(L.c1)[r] = c1;
      gmut<float>(L.c2)[r] = c2;
    }
    row_slices<VEC>(L.ld, [&](int c, auto whole, int n) {
      constexpr bool kWhole = decltype(whole)::value;
      float h[VEC], dy[VEC], g[VEC], d[VEC] = {};
      ln_input<T, VEC, kWhole>(L, base, c, n, h);
      slice_in<T, VEC, kWhole>(static_cast<const T*>(L.dy), base + c, n, dy);
      slice_in<float, VEC, kWhole>(L.gamma, c, n, g);
      if (L.dsum) slice_in<T, VEC, kWhole>(static_cast<const T*>(L.dsum), base + c, n, d);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        h[e] = rs * __builtin_fmaf(-((h[e] - mu) * rs), c1, dy[e] * g[e] - c2) + d[e];
      slice_out<T, VEC, kWhole>(L.out, base + c, n, h);
    });
  }
}

// Column sums of long rows, from dy and x once more (bound by memory): eight columns per lane (fp32 four), every (4 gridDim.y)-th row per wave, the four waves'
// sums through LDS.
template <typename T>
__global__ __launch_bounds__(256) void ln_backward_columns_kernel(const LnTrain L) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ float s_sum[4][64 * kVec];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * kVec;
  const int live = (int)min((int64_t)kVec, max((int64_t)L.ld - c, (int64_t)0));
  float sg[kVec] = {}, sb[kVec] = {}, sh[kVec] = {}, g[kVec] = {}, bi[kVec] = {};
#pragma unroll
  for (int e = 0; e < kVec; ++e)
    if (e < live) {
      g[e] = gconst<float>(L.gamma)[c + e];
      if (L.bias) bi[e] = gconst<float>(L.bias)[c + e];
    }
  auto some = [&](const void* p, int64_t at) {
    Pack<T, kVec> v{};
    if (live == kVec) {
      v = load_slice<T, kVec>(gconst<T>(p) + at);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e < live) v.v[e] = gconst<T>(p)[at + e];
    }
    return v;
  };
  if (live > 0)
    for (int64_t r = blockIdx.y * 4 + wave; r < L.rows; r += 4 * gridDim.y) {
      const int64_t at = r * L.ld + c;
      const float mu = gconst<float>(L.mean)[r], rs = gconst<float>(L.rstd)[r];
      const float c1 = gconst<float>(L.c1)[r], c2 = gconst<float>(L.c2)[r];
      const Pack<T, kVec> dy = some(L.dy, at), x = some(L.x, at);
      Pack<T, kVec> s{}, d{};
      if (L.skip) s = some(L.skip, at);
      if (L.part_bias && L.dsum) d = some(L.dsum, at);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        float h = (float)x.v[e];
        if (L.skip) h += (float)s.v[e];
        h += bi[e];
        const float w = (float)dy.v[e], xh = (h - mu) * rs;
        sg[e] = __builtin_fmaf(w, xh, sg[e]);
        sb[e] += w;
        sh[e] += rs * __builtin_fmaf(-xh, c1, w * g[e] - c2) + (float)d.v[e];
      }
    }
  auto leave = [&](const float (&v)[kVec], float* part) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kVec; ++e) s_sum[wave][lane * kVec + e] = v[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * kVec; i += 256) {
      const int64_t col = (int64_t)blockIdx.x * 64 * kVec + i;
      if (col < L.ld)
        gmut<float>(part)[blockIdx.y * L.part_stride + col] = ((s_sum[0][i] + s_sum[1][i]) + s_sum[2][i]) + s_sum[3][i];
    }
  };
  leave(sg, L.part_gamma);
  leave(sb, L.part_beta);
  if (L.part_bias) leave(sh, L.part_bias);
}

// ---- launch ---------------------------------------------------------------------------------------------------

constexpr int kMaxParts = 256;       // rows of partials a backward launch leaves (its workgroups)
constexpr int kLongParts = 32;       // the same for long rows, whose column sums are a launch of their own
constexpr int kBackwardWG = 512;
// Lanes of a backward workgroup (one per CU) that sums columns in registers.  Rows of 256 lanes with one slice each have few
// bytes in flight and registers for twice the lanes: 8192 x 2048 fp16 24.3 us for 26.6, 4099 x 1531 16.5 for 17.8.  With
// 64 lanes it is no gain (4099 x 509 9.1 for 8.4, 20000 x 300 15.8 for 16.9), and two fp32 slices spill.
constexpr int sums_wg(int vec, int nv, int lpr) { return vec == 8 && nv == 1 && lpr == 256 ? 1024 : kBackwardWG; }

// Lanes per row and steps per lane of a row of `ld` elements in slices of VEC; steps == 0: streamed.
struct Shape {
  int lpr, nv;
};
Shape row_shape(int ld, int vec) {
  const int64_t slices = ((int64_t)ld + vec - 1) / vec;
  if (slices <= 8) return {8, 1};
  if (slices <= 16) return {16, 1};
  if (slices <= 32) return {32, 1};
  const int deep = 16 / vec;  // steps that keep 16 elements per lane
  for (int nv = 1; nv <= deep; nv *= 2)
    if (slices <= 64 * nv) return {64, nv};
  for (int nv = 1; nv <= deep; nv *= 2)
    if (slices <= 256 * nv) return {256, nv};
  if (slices <= 512 * deep) return {512, deep};
  // fp32 rows of more than 16 elements per lane do not fit its registers: 2700 x 12288 took 124 us forward and 275 us
  // backward that way, 74 and 146 streamed (a row of up to some 40000 elements would fit LDS, which is not tried)
  if (vec == 8 && slices <= 1024 * deep) return {512, 2 * deep};
  return {0, 0};
}

// Calls f with std::true_type for a row that fills every lane.  (Rows of a few single elements have fewer than lanes.)
template <int VEC, int NV, int LPR, typename F>
void with_full(int ld, F&& f) {
  if constexpr (VEC > 1) {
    if (ld == LPR * VEC * NV) return f(std::true_type{});
  }
  f(std::false_type{});
}

template <typename T, int VEC, int NV, int LPR>
int launch_forward(const LnTrain& L, hipStream_t stream) {
  constexpr int kWG = LPR <= 256 ? 256 : 512;
  constexpr int kRows = kWG / LPR;
  const int64_t want = (L.rows + kRows - 1) / kRows;
  const unsigned grid = (unsigned)std::min<int64_t>(want, (int64_t)device_cus() * (kWG == 256 ? 4 : 2));
  with_full<VEC, NV, LPR>(L.ld, [&](auto full) {
    hipLaunchKernelGGL((ln_forward_kernel<T, VEC, NV, kWG, LPR, decltype(full)::value>), dim3(grid), dim3(kWG), 0, stream, L);
  });
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

template <typename T, int VEC, int NV, int LPR>
int launch_backward(const LnTrain& L, unsigned grid, hipStream_t stream) {
  constexpr bool kSums = NV * VEC <= 16;
  const bool columns = (int)grid > L.row_blocks;  // workgroups that sum columns
  with_full<VEC, NV, LPR>(L.ld, [&](auto full) {
    auto launch = [&](auto bias, auto sums) {
      constexpr int kWG = decltype(sums)::value ? sums_wg(VEC, NV, LPR) : kBackwardWG;
      hipLaunchKernelGGL((ln_backward_kernel<T, VEC, NV, kWG, LPR, decltype(full)::value, decltype(bias)::value,
                                             decltype(sums)::value>),
                         dim3(grid), dim3(kWG), 0, stream, L);
    };
    if (columns)
      launch(std::false_type{}, std::false_type{});
    else if (L.bias)
      launch(std::true_type{}, std::integral_constant<bool, kSums>{});
    else
      launch(std::false_type{}, std::integral_constant<bool, kSums>{});
  });
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

// Calls f.template operator()<VEC, NV, LPR>() for the row's shape; false where rows are streamed.
template <typename T, typename F>
bool with_shape(int ld, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kDeep = 16 / kVec;
  if (ld < kVec) {
    f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
    return true;
  }
  const Shape s = row_shape(ld, kVec);
  using V = std::integral_constant<int, kVec>;
#define FWDMI_SHAPE(LPR_, NV_)                                                                       \
  if (s.lpr == LPR_ && s.nv == NV_) {                                                                \
    f(V{}, std::integral_constant<int, NV_>{}, std::integral_constant<int, LPR_>{});                 \
    return true;                                                                                     \
  }
  FWDMI_SHAPE(8, 1)
  FWDMI_SHAPE(16, 1)
  FWDMI_SHAPE(32, 1)
  FWDMI_SHAPE(64, 1)
  FWDMI_SHAPE(64, 2)
  FWDMI_SHAPE(256, 2)
  if constexpr (kDeep == 2) {
    FWDMI_SHAPE(256, 1)
  } else {
    FWDMI_SHAPE(64, 4)
    FWDMI_SHAPE(256, 4)
  }
  FWDMI_SHAPE(512, kDeep)
  if constexpr (kVec == 8) {
    FWDMI_SHAPE(512, 2 * kDeep)
  }
#undef FWDMI_SHAPE
  return false;
}

constexpr int32_t kMaxLd = 1 << 26;  // the launch that adds partials holds 16 work-items per column of each of three sums

// Rows of more than 16 elements per lane, or streamed: column sums by ln_backward_columns_kernel.
bool long_rows(int ld, int dtype) {
  const int vec = dtype == FWDMI_F32 ? 4 : 8;
  if (ld < vec) return false;
  const Shape s = row_shape(ld, vec);
  return s.lpr == 0 || s.nv * vec > 16;
}

// Workgroups of rows of a backward call with column sums in registers, or with workgroups for them.
int64_t row_groups(int ld, int64_t rows, int dtype, bool joint) {
  const int vec = dtype == FWDMI_F32 ? 4 : 8;
  const Shape s = ld < vec ? Shape{8, 1} : row_shape(ld, vec);
  const int per = (joint ? kBackwardWG : sums_wg(vec, s.nv, s.lpr)) / s.lpr;
  return (rows + per - 1) / per;
}

// Few rows of more than one workgroup, no bias: rows and column sums in one launch (509 x 768 fp32: 6 us; 5 and 3 us in
// two launches, and 5 us less on the host).
constexpr int64_t kFewRows = 1024;
bool joint_rows(int ld, int64_t rows, int dtype, bool bias) {
  return !bias && rows <= kFewRows && !long_rows(ld, dtype) && row_groups(ld, rows, dtype, true) > 1;
}

// Rows of partials of a backward call.
int64_t backward_parts(int ld, int64_t rows, int dtype, bool bias) {
  if (rows == 0 || joint_rows(ld, rows, dtype, bias)) return 0;
  if (long_rows(ld, dtype)) return std::min<int64_t>((rows + 3) / 4, kLongParts);
  return std::min<int64_t>(row_groups(ld, rows, dtype, false), kMaxParts);
}

template <typename T>
int forward_typed(const LnTrain& L, hipStream_t stream) {
  int rc = FWDMI_OK;
  const bool done = with_shape<T>(L.ld, [&](auto vec, auto nv, auto lpr) {
    rc = launch_forward<T, decltype(vec)::value, decltype(nv)::value, decltype(lpr)::value>(L, stream);
  });
  if (done) return rc;
  const unsigned grid = (unsigned)std::min<int64_t>(L.rows, (int64_t)device_cus() * 4);
  hipLaunchKernelGGL((ln_forward_stream_kernel<T>), dim3(grid), dim3(kStreamWG), 0, stream, L);
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

template <typename T>
int backward_typed(LnTrain& L, int64_t parts, bool long_row, hipStream_t stream) {
  int rc = FWDMI_OK;
  int64_t grid = parts;
  if (parts == 0) {
    const int dtype = sizeof(T) == 4 ? FWDMI_F32 : FWDMI_F16;
    L.row_blocks = (int)row_groups(L.ld, L.rows, dtype, true);
    grid = L.row_blocks + ((int64_t)L.ld + 63) / 64;
  } else {
    if (long_row) grid = std::min<int64_t>(L.rows, (int64_t)device_cus() * 2);
    L.row_blocks = (int)grid;
  }
  const bool done = with_shape<T>(L.ld, [&](auto vec, auto nv, auto lpr) {
    rc = launch_backward<T, decltype(vec)::value, decltype(nv)::value, decltype(lpr)::value>(L, (unsigned)grid, stream);
  });
  if (!done) {
    hipLaunchKernelGGL((ln_backward_stream_kernel<T>), dim3((unsigned)grid), dim3(kStreamWG), 0, stream, L);
    FWDMI_HIP_CHECK(hipGetLastError());
  }
  if (rc != FWDMI_OK || !long_row) return rc;
  constexpr int kColumns = 64 * 16 / (int)sizeof(T);
  const dim3 cgrid((unsigned)(((int64_t)L.ld + kColumns - 1) / kColumns), (unsigned)parts);
  hipLaunchKernelGGL((ln_backward_columns_kernel<T>), cgrid, dim3(256), 0, stream, L);
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

}  // namespace
}  // namespace fwdmi

extern "C" {

int fwdmi_layer_norm_forward(void* stream, int32_t ld, int64_t n, const void* x, const void* skip, const float* beta,
                             const float* gamma, const float* bias, void* y, void* sum, float* mean, float* rstd,
                             int32_t dtype, float eps) {
  using namespace fwdmi;
  clear_error();
  if (!is_train_dtype(dtype)) return set_error(FWDMI_ERR_UNSUPPORTED, "layer norm forward: unsupported dtype %d", dtype);
  FWDMI_REQUIRE(ld > 0 && ld <= kMaxLd && n >= 0 && n % ld == 0,
                "layer norm forward: n=%lld is not a multiple of ld=%d (at most 2^26)", (long long)n, ld);
  if (n == 0) return FWDMI_OK;
  FWDMI_REQUIRE(x && beta && gamma && y && mean && rstd, "layer norm forward: null pointer");
  LnTrain L{};
  L.x = x;
  L.skip = skip;
  L.gamma = gamma;
  L.beta = beta;
  L.bias = bias;
  L.out = y;
  L.sum = sum;
  L.mean = mean;
  L.rstd = rstd;
  L.rows = n / ld;
  L.ld = ld;
  L.eps = eps;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FWDMI_F16) return forward_typed<_Float16>(L, s);
  if (dtype == FWDMI_BF16) return forward_typed<__bf16>(L, s);
  return forward_typed<float>(L, s);
}

size_t fwdmi_layer_norm_backward_workspace(int32_t ld, int64_t n, int32_t with_bias, int32_t dtype) {
  using namespace fwdmi;
  if (!is_train_dtype(dtype) || ld <= 0 || ld > kMaxLd || n <= 0 || n % ld != 0) return 0;
  const int64_t rows = n / ld;
  const int64_t parts = backward_parts(ld, rows, dtype, with_bias != 0);
  size_t bytes = parts > 1 ? (size_t)parts * (with_bias ? 3 : 2) * (size_t)ld * sizeof(float) : 0;
  if (long_rows(ld, dtype)) bytes += (size_t)rows * 2 * sizeof(float);
  return bytes;
}

int fwdmi_layer_norm_backward(void* stream, int32_t ld, int64_t n, const void* dy, const void* x, const void* skip,
                              const void* dsum, const float* gamma, const float* bias, const float* mean,
                              const float* rstd, void* dx, float* dgamma, float* dbeta, float* dbias, void* workspace,
                              size_t workspace_size, int32_t dtype) {
  using namespace fwdmi;
  clear_error();
  if (!is_train_dtype(dtype)) return set_error(FWDMI_ERR_UNSUPPORTED, "layer norm backward: unsupported dtype %d", dtype);
  FWDMI_REQUIRE(ld > 0 && ld <= kMaxLd && n >= 0 && n % ld == 0,
                "layer norm backward: n=%lld is not a multiple of ld=%d (at most 2^26)", (long long)n, ld);
  FWDMI_REQUIRE(dgamma && dbeta && (bias == nullptr) == (dbias == nullptr),
                "layer norm backward: dgamma and dbeta are written always, dbias exactly where there is a bias");
  const int64_t rows = n / ld;
  const int kinds = bias ? 3 : 2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t parts = backward_parts(ld, rows, dtype, bias != nullptr);
  LnTrain L{};
  if (rows > 0) {
    FWDMI_REQUIRE(dy && x && gamma && mean && rstd && dx, "layer norm backward: null pointer");
    const size_t need = fwdmi_layer_norm_backward_workspace(ld, n, bias != nullptr, dtype);
    FWDMI_REQUIRE(need == 0 || (workspace && workspace_size >= need && reinterpret_cast<uintptr_t>(workspace) % 4 == 0),
                  "layer norm backward: workspace of %zu bytes, %zu needed", workspace ? workspace_size : (size_t)0, need);
    L.dy = dy;
    L.x = x;
    L.skip = skip;
    L.dsum = dsum;
    L.gamma = gamma;
    L.bias = bias;
    L.mean = const_cast<float*>(mean);
    L.rstd = const_cast<float*>(rstd);
    L.out = dx;
    L.rows = rows;
    L.ld = ld;
    float* const ws = static_cast<float*>(workspace);
    const bool long_row = long_rows(ld, dtype);
    if (long_row) {
      L.c1 = ws + (parts > 1 ? parts * kinds * (int64_t)ld : 0);
      L.c2 = L.c1 + rows;
    }
    if (parts <= 1) {  // one workgroup's sums are the result, or the columns' own
      L.part_gamma = dgamma;
      L.part_beta = dbeta;
      L.part_bias = dbias;
    } else {
      L.part_gamma = ws;
      L.part_beta = ws + ld;
      L.part_bias = bias ? ws + 2 * (int64_t)ld : nullptr;
      L.part_stride = (int64_t)kinds * ld;
    }
    const int rc = dtype == FWDMI_F16    ? backward_typed<_Float16>(L, parts, long_row, s)
                   : dtype == FWDMI_BF16 ? backward_typed<__bf16>(L, parts, long_row, s)
                                         : backward_typed<float>(L, parts, long_row, s);
    if (rc != FWDMI_OK || parts <= 1) return rc;
  }
  ColumnSums S{};
  S.part = static_cast<const float*>(workspace);
  S.out[0] = dgamma;
  S.out[1] = dbeta;
  S.out[2] = dbias;
  S.parts = (int32_t)parts;
  S.ld = ld;
  S.kinds = kinds;
  return launch_column_sums(S, s);
}

}  // extern "C"
