// Rows over threads: what the norm kernels share.  A thread holds units of 8
// consecutive columns.  WARP: rows of at most 1024 columns belong to a warp, 8 to a
// block, and need no barrier; longer ones to a block.
#pragma once

#include "checkpoint8.cuh"

namespace mhc {
namespace {

constexpr int kWarpCols = 1024, kWarpRows = 8;

// Sum over the row's threads, the same in each.
template <bool WARP>
__device__ __forceinline__ float row_total(float v, float* red) {
  v = warp_sum(v);
  if (WARP) return v;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nw ? red[lane] : 0.f);
}
// Column of a thread's unit k, of the first unit of its warp
template <bool WARP>
__device__ __forceinline__ int64_t unit_col(int k) {
  return 8 * (WARP ? (int64_t)(k * 32 + (threadIdx.x & 31)) : (int64_t)k * blockDim.x + threadIdx.x);
}

// Eight weights; columns past the end read as zero
__device__ __forceinline__ void load_w(const float* w, int64_t c, int64_t cols, float (&v)[8]) {
  if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(w) & 31) == 0) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(w + c)), b = __ldg(reinterpret_cast<const float4*>(w + c + 4));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? __ldg(w + c + j) : 0.f;
  }
}

// Units of rows that wide accesses do not fit, types by a branch
__device__ __forceinline__ void load_any(const void* p, bool b16, int64_t row, int64_t c, int64_t cols, float* mine, float (&v)[8]) {
  const int64_t c0 = c - 8 * (threadIdx.x & 31);
  if (b16) ck_load_any(static_cast<const __nv_bfloat16*>(p) + row * cols, c0, cols, mine, v);
  else ck_load_any(static_cast<const float*>(p) + row * cols, c0, cols, mine, v);
}
__device__ __forceinline__ void save_any(void* p, bool b16, int64_t row, int64_t c, int64_t cols, float* mine, const float (&v)[8]) {
  const int64_t c0 = c - 8 * (threadIdx.x & 31);
  if (b16) ck_save_any(static_cast<__nv_bfloat16*>(p) + row * cols, c0, cols, mine, v);
  else ck_save_any(static_cast<float*>(p) + row * cols, c0, cols, mine, v);
}

template <typename T>
bool even_rows(const void* p, int64_t cols, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & (8 * sizeof(T) - 1)) == 0 && cols % 8 == 0 && stride % 8 == 0;
}

}  // namespace
}  // namespace mhc
