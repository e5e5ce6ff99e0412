// Slices of a few elements at any element alignment, and the sum of partial rows: shared by the training and linear
// kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>

#include "../common.h"
#include "device_util.h"

namespace fwdmi {
namespace {

// N elements at any element alignment (one global_load_dwordx4 where the slice is 16 bytes).
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_slice(const T FWDMI_GLOBAL* p) {
  Pack<T, N> r;
  if constexpr (N == 1) {
    r.v[0] = *p;
  } else {
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    const V x = *(const V FWDMI_GLOBAL*)p;
    __builtin_memcpy(&r, &x, sizeof(r));
  }
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_slice(T FWDMI_GLOBAL* p, const Pack<T, N>& r) {
  if constexpr (N == 1) {
    *p = r.v[0];
  } else {
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    V x;
    __builtin_memcpy(&x, &r, sizeof(r));
    *(V FWDMI_GLOBAL*)p = x;
  }
}

// The sum over `rows` rows of column c (64 columns per workgroup, one per lane), in a fixed order: each of the WAVES waves
// adds every WAVES-th row, eight in flight, wave 0 adds the waves' sums and returns it.
template <typename T, int WAVES>
__device__ __forceinline__ float column_sum(const T* part, int64_t rows, int64_t width, int64_t c, float (*s_red)[64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float a = 0.0f;
  if (c < width) {
    const T FWDMI_GLOBAL* at = gconst<T>(part) + wave * width + c;
    int64_t left = (rows - wave + WAVES - 1) / WAVES;  // rows of this wave
    for (; left >= 8; left -= 8, at += 8 * WAVES * width) {
      T v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = at[k * WAVES * width];
#pragma unroll
      for (int k = 0; k < 8; ++k) a += (float)v[k];
    }
    for (; left > 0; --left, at += WAVES * width) a += (float)*at;
  }
  s_red[wave][lane] = a;
  __syncthreads();
  if (wave == 0)
    for (int k = 1; k < WAVES; ++k) a += s_red[k][lane];
  return a;
}

// Adds `parts` rows of partials; parts == 0 leaves zeros.  A launch's own cost and one pass of memory latency: 256 rows of
// 2 x 1024 sums (2 MB) take 3.9 us, of which an empty launch is 2.
struct ColumnSums {
  const float* part;  // [parts][kinds * ld]
  float* out[3];      // [ld] each
  int32_t parts, ld, kinds;
};
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(64 * kSumWaves) void column_sums_kernel(const ColumnSums S) {
  __shared__ float s_red[kSumWaves][64];
  const int64_t width = (int64_t)S.kinds * S.ld, c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float a = column_sum<float, kSumWaves>(S.part, S.parts, width, c, s_red);
  if (threadIdx.x < 64 && c < width) {
    const int kind = (int)(c / S.ld);
    float* const out = kind == 0 ? S.out[0] : kind == 1 ? S.out[1] : S.out[2];
    gmut<float>(out)[c - (int64_t)kind * S.ld] = a;
  }
}

// A launch holds fewer than 2^32 work-items.
inline bool launchable(int64_t workgroups, int threads) { return workgroups <= 0xffffffffll / threads; }
inline int check_launch(int64_t workgroups, int threads) {
  if (launchable(workgroups, threads)) return FWDMI_OK;
  return set_error(FWDMI_ERR_UNSUPPORTED, "a launch of %lld workgroups of %d", (long long)workgroups, threads);
}

inline int launch_column_sums(const ColumnSums& S, hipStream_t stream) {
  const int64_t grid = ((int64_t)S.kinds * S.ld + 63) / 64;
  if (const int rc = check_launch(grid, 64 * kSumWaves)) return rc;
  hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)grid), dim3(64 * kSumWaves), 0, stream, S);
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

// Compute units of the current device (asked once per device).
inline int device_cus() {
  static std::atomic<int> known[64];
  int dev = 0, v = 0;
  if (hipGetDevice(&dev) == hipSuccess) {
    const bool keep = dev >= 0 && dev < 64;
    if (keep && (v = known[dev].load(std::memory_order_relaxed)) > 0) return v;
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0) {
      if (keep) known[dev].store(v, std::memory_order_relaxed);
      return v;
    }
  }
  (void)hipGetLastError();
  return 256;
}

// Types of the training and linear launchers.
inline bool is_train_dtype(int t) { return t == FWDMI_F32 || t == FWDMI_F16 || t == FWDMI_BF16; }

}  // namespace
}  // namespace fwdmi
