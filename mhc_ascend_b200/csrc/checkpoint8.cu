// 8-bit activation checkpoints: pack, restore, and RMSNorm that keeps its
// input in 8 bits (forward and backward).  Format: checkpoint8.cuh.
#include "checkpoint8.cuh"

namespace mhc {
namespace {

// Row and unit (of V columns) of a flat unit index, stepped without divisions.
struct UnitWalk {
  int64_t row;
  int64_t u;
  __device__ __forceinline__ UnitWalk(int64_t i, int64_t U) : row(i / U), u(i % U) {}
  __device__ __forceinline__ void step(int64_t drow, int64_t du, int64_t U) {
    row += drow;
    u += du;
    if (u >= U) { u -= U; ++row; }
  }
};

// ---------------------------------------------------------------------------
// pack / unpack: one pass, bound by HBM.  A thread takes units of 8 columns
// (32 or 16 bytes in, 8 bytes of codes out), kUnroll of them so that enough
// loads are in flight.  Rows whose start or width breaks 16-byte accesses take
// one column per lane instead (a block is then a warp).
// ---------------------------------------------------------------------------
constexpr int kPackThreads = 256, kUnroll = 4;

template <typename T, int V>
__global__ void __launch_bounds__(kPackThreads)
    pack_kernel(const T* __restrict__ x, int64_t stride, int8_t* __restrict__ codes,
                uint8_t* __restrict__ exps, int64_t rows, int64_t cols, int64_t U) {
  const int64_t pitch = U * V, total = rows * U;
  const int64_t first = (int64_t)blockIdx.x * (kPackThreads * kUnroll) + threadIdx.x;
  const int64_t drow = kPackThreads / U, du = kPackThreads % U;
  UnitWalk at(first, U);
  float v[kUnroll][V];
  int64_t row[kUnroll], col[kUnroll];
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    row[k] = at.row;
    col[k] = at.u * V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[k][j] = 0.f;
    if (at.row < rows && col[k] < cols) {  // V = 8: cols % 8 == 0, so a unit lies in the row or past it
      ck_load(x + at.row * stride + col[k], v[k]);
    }
    at.step(drow, du, U);
  }
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    const bool on = first + (int64_t)k * kPackThreads < total;
    ck_encode<V>(v[k], codes + row[k] * pitch, exps + row[k] * (pitch / kCkBlock), col[k], on);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kPackThreads)
    unpack_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                  T* __restrict__ out, int64_t rows, int64_t cols, int64_t U, int64_t pitch) {
  const int64_t first = (int64_t)blockIdx.x * (kPackThreads * kUnroll) + threadIdx.x;
  const int64_t drow = kPackThreads / U, du = kPackThreads % U;
  UnitWalk at(first, U);
  float v[kUnroll][V];
  int64_t row[kUnroll], col[kUnroll];
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    row[k] = at.row;
    col[k] = at.u * V;
    if (at.row < rows && col[k] < cols)
      ck_decode<V>(codes + at.row * pitch, exps + at.row * (pitch / kCkBlock), col[k], v[k]);
    at.step(drow, du, U);
  }
#pragma unroll
  for (int k = 0; k < kUnroll; ++k)
    if (row[k] < rows && col[k] < cols) ck_save(out + row[k] * cols + col[k], v[k]);
}

// ---------------------------------------------------------------------------
// RMSNorm.  r = sqrt(mean x^2 + eps), y = x / r * w, and the codes of x, in one
// pass over x: a row stays in its block's registers between the sum and the
// output (UPT units of V columns a thread).
// ---------------------------------------------------------------------------
__device__ __forceinline__ float block_total(float v, float* red) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < nw; ++w) s += red[w];
  return s;
}

// Most threads of a block by the share of a row that one thread holds: more
// than 512 only where the largest share needs them.
constexpr int row_threads(int V, int UPT) { return UPT == (V == 8 ? 4 : 16) ? 1024 : 512; }

template <typename T, int V, int UPT>
__global__ void __launch_bounds__(row_threads(V, UPT))
    norm_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w, T* __restrict__ out,
                    float* __restrict__ rms, int8_t* __restrict__ codes, uint8_t* __restrict__ exps,
                    int64_t cols, int64_t pitch, float eps) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * cols;
  float v[UPT][V];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = ((int64_t)k * blockDim.x + threadIdx.x) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[k][j] = 0.f;
    if (c < cols) ck_load(xr + c, v[k]);
  }
#pragma unroll
  for (int k = 0; k < UPT; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fmaf(v[k][j], v[k][j], ss);
  const float r = sqrtf(block_total(ss, red) / (float)cols + eps);
  const float ir = 1.0f / r;
  if (threadIdx.x == 0) rms[row] = r;
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = ((int64_t)k * blockDim.x + threadIdx.x) * V;
    if (c < cols) {
      float o[V], wv[V];
      ck_load(w + c, wv);
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = v[k][j] * ir * wv[j];
      ck_save(out + row * cols + c, o);
    }
    ck_encode<V>(v[k], codes + row * pitch, exps + row * (pitch / kCkBlock), c, c < pitch);
  }
}

// Rows too long for registers: the row is read twice (the second time from L2).
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_fwd_long_kernel(const T* __restrict__ x, const float* __restrict__ w, T* __restrict__ out,
                         float* __restrict__ rms, int8_t* __restrict__ codes, uint8_t* __restrict__ exps,
                         int64_t cols, int64_t pitch, float eps) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * cols;
  float ss = 0.f;
  for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
    const float t = ck_f32(xr[c]);
    ss = fmaf(t, t, ss);
  }
  const float r = sqrtf(block_total(ss, red) / (float)cols + eps);
  const float ir = 1.0f / r;
  if (threadIdx.x == 0) rms[row] = r;
  for (int64_t c = threadIdx.x; c - threadIdx.x < pitch; c += blockDim.x) {
    float v[1] = {c < cols ? ck_f32(xr[c]) : 0.f};
    if (c < cols) ck_store(out + row * cols + c, v[0] * ir * w[c]);
    ck_encode<1>(v, codes + row * pitch, exps + row * (pitch / kCkBlock), c, c < pitch);
  }
}

// Backward at the restored input xh:
//   gx = (g w - xh * D / (cols r^2)) / r,  D = sum_c g w xh
//   gw = sum over rows of g xh / r
// A block walks rows blockIdx.x, + gridDim.x, ...; its threads keep their
// columns' share of gw in registers over all of them, so g and the codes are
// read once and gw leaves as one row of partial sums a block, added in block
// order by norm_gw_kernel: no atomics, the same bits every time.
template <typename T, int V, int UPT>
__global__ void __launch_bounds__(row_threads(V, UPT))
    norm_bwd_kernel(const T* __restrict__ g, const int8_t* __restrict__ codes,
                    const uint8_t* __restrict__ exps, const float* __restrict__ w,
                    const float* __restrict__ rms, T* __restrict__ gx, float* __restrict__ part,
                    int64_t rows, int64_t cols, int64_t pitch) {
  __shared__ float red[2][32];
  float acc[UPT][V];
#pragma unroll
  for (int k = 0; k < UPT; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) acc[k][j] = 0.f;
  int buf = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, buf ^= 1) {
    float gv[UPT][V], xv[UPT][V];
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int64_t c = ((int64_t)k * blockDim.x + threadIdx.x) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) gv[k][j] = xv[k][j] = 0.f;
      if (c < cols) {
        ck_load(g + row * cols + c, gv[k]);
        ck_decode<V>(codes + row * pitch, exps + row * (pitch / kCkBlock), c, xv[k]);
      }
    }
    const float r = rms[row], ir = 1.0f / r;
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int64_t c = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      float wv[V];
      if (c < cols) {
        ck_load(w + c, wv);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          acc[k][j] = fmaf(gv[k][j] * ir, xv[k][j], acc[k][j]);
          gv[k][j] *= wv[j];
          d = fmaf(gv[k][j], xv[k][j], d);
        }
      }
    }
    // two buffers: a block writes red[buf] again only after the barrier of the row between
    const float coef = block_total(d, red[buf]) / ((float)cols * r * r);
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int64_t c = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      if (c < cols) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (gv[k][j] - xv[k][j] * coef) * ir;
        ck_save(gx + row * cols + c, o);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = ((int64_t)k * blockDim.x + threadIdx.x) * V;
    if (c < cols) {
      float* p = part + (int64_t)blockIdx.x * cols + c;
#pragma unroll
      for (int j = 0; j < V; ++j) p[j] = acc[k][j];
    }
  }
}

// Long rows: two passes a row, gw added up in the block's own row of partials.
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_bwd_long_kernel(const T* __restrict__ g, const int8_t* __restrict__ codes,
                         const uint8_t* __restrict__ exps, const float* __restrict__ w,
                         const float* __restrict__ rms, T* __restrict__ gx, float* __restrict__ part,
                         int64_t rows, int64_t cols, int64_t pitch) {
  __shared__ float red[2][32];
  float* p = part + (int64_t)blockIdx.x * cols;
  for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) p[c] = 0.f;
  int buf = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, buf ^= 1) {
    const int8_t* cr = codes + row * pitch;
    const uint8_t* er = exps + row * (pitch / kCkBlock);
    const T* gr = g + row * cols;
    const float r = rms[row], ir = 1.0f / r;
    float d = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float xv[1];
      ck_decode<1>(cr, er, c, xv);
      const float gv = ck_f32(gr[c]);
      p[c] = fmaf(gv * ir, xv[0], p[c]);
      d = fmaf(gv * w[c], xv[0], d);
    }
    const float coef = block_total(d, red[buf]) / ((float)cols * r * r);
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float xv[1];
      ck_decode<1>(cr, er, c, xv);
      ck_store(gx + row * cols + c, (ck_f32(gr[c]) * w[c] - xv[0] * coef) * ir);
    }
  }
}

// gw[c] = sum of part[0..blocks)[c]: 32 columns a block, 8 threads a column,
// each a fixed share of the partial rows.
__global__ void __launch_bounds__(256)
    norm_gw_kernel(const float* __restrict__ part, float* __restrict__ gw, int blocks, int64_t cols) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int b = q; b < blocks; b += 8) t += part[(int64_t)b * cols + c];
  s[q][lane] = t;
  __syncthreads();
  if (q == 0 && c < cols) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) a += s[k][lane];
    gw[c] = a;
  }
}

// How a row of `cols` columns is laid over a block: V columns a unit, UPT units
// a thread, `threads` threads; UPT = 0: the row does not fit the registers.
struct RowPlan {
  int V, UPT, threads;
};
RowPlan row_plan(int64_t cols, bool vec) {
  const int64_t U = vec ? ck_pitch(cols) / 8 : ck_pitch(cols);
  const int cand[3] = {1, 2, 4};
  const int wide[4] = {1, 4, 8, 16};
  if (vec) {
    for (int upt : cand) {
      const int64_t th = (((U + upt - 1) / upt) + 31) / 32 * 32;
      if (th <= row_threads(8, upt)) return {8, upt, (int)th};
    }
  } else {
    for (int upt : wide) {
      const int64_t th = (((U + upt - 1) / upt) + 31) / 32 * 32;
      if (th <= row_threads(1, upt)) return {1, upt, (int)th};
    }
  }
  return {1, 0, 1024};
}

template <typename T>
bool vec_ok(const void* p, int64_t cols, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & (8 * sizeof(T) - 1)) == 0 && cols % 8 == 0 && stride % 8 == 0;
}

template <typename T>
int launch_pack(const T* x, int64_t stride, int8_t* codes, uint8_t* exps, int64_t rows, int64_t cols,
                cudaStream_t st) {
  const bool vec = vec_ok<T>(x, cols, stride);
  const int64_t U = ck_pitch(cols) / (vec ? 8 : 1);
  const int64_t blocks = (rows * U + kPackThreads * kUnroll - 1) / (kPackThreads * kUnroll);
  MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "checkpoint8_pack: %lld x %lld values are too many",
              (long long)rows, (long long)cols);
  ProfScope p("checkpoint8_pack", st);
  if (vec) pack_kernel<T, 8><<<(unsigned)blocks, kPackThreads, 0, st>>>(x, stride, codes, exps, rows, cols, U);
  else pack_kernel<T, 1><<<(unsigned)blocks, kPackThreads, 0, st>>>(x, stride, codes, exps, rows, cols, U);
  return check_launch("checkpoint8_pack");
}

template <typename T>
int launch_unpack(const int8_t* codes, const uint8_t* exps, T* out, int64_t rows, int64_t cols, cudaStream_t st) {
  const bool vec = vec_ok<T>(out, cols, cols);
  const int64_t U = (cols + (vec ? 7 : 0)) / (vec ? 8 : 1);
  const int64_t blocks = (rows * U + kPackThreads * kUnroll - 1) / (kPackThreads * kUnroll);
  MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "checkpoint8_unpack: %lld x %lld values are too many",
              (long long)rows, (long long)cols);
  ProfScope p("checkpoint8_unpack", st);
  const int64_t pitch = ck_pitch(cols);
  if (vec) unpack_kernel<T, 8><<<(unsigned)blocks, kPackThreads, 0, st>>>(codes, exps, out, rows, cols, U, pitch);
  else unpack_kernel<T, 1><<<(unsigned)blocks, kPackThreads, 0, st>>>(codes, exps, out, rows, cols, U, pitch);
  return check_launch("checkpoint8_unpack");
}

template <typename T>
int launch_norm_fwd(const T* x, const float* w, T* out, float* rms, int8_t* codes, uint8_t* exps, int64_t rows,
                    int64_t cols, float eps, cudaStream_t st) {
  const bool vec = vec_ok<T>(x, cols, cols) && vec_ok<T>(out, cols, cols) && vec_ok<float>(w, cols, cols);
  const RowPlan pl = row_plan(cols, vec);
  const int64_t pitch = ck_pitch(cols);
  ProfScope p("rmsnorm_checkpoint8_fwd", st);
#define MHC_NORM_FWD(VV, UU) \
  norm_fwd_kernel<T, VV, UU><<<(unsigned)rows, pl.threads, 0, st>>>(x, w, out, rms, codes, exps, cols, pitch, eps)
  if (pl.UPT == 0)
    norm_fwd_long_kernel<T><<<(unsigned)rows, pl.threads, 0, st>>>(x, w, out, rms, codes, exps, cols, pitch, eps);
  else if (pl.V == 8 && pl.UPT == 1) MHC_NORM_FWD(8, 1);
  else if (pl.V == 8 && pl.UPT == 2) MHC_NORM_FWD(8, 2);
  else if (pl.V == 8) MHC_NORM_FWD(8, 4);
  else if (pl.UPT == 1) MHC_NORM_FWD(1, 1);
  else if (pl.UPT == 4) MHC_NORM_FWD(1, 4);
  else if (pl.UPT == 8) MHC_NORM_FWD(1, 8);
  else MHC_NORM_FWD(1, 16);
#undef MHC_NORM_FWD
  return check_launch("rmsnorm_checkpoint8_fwd");
}

int norm_bwd_blocks(int64_t rows, int64_t cols) {
  // two blocks an SM at most; fewer rows than that: one block a row
  const int64_t most = 2 * (int64_t)num_sms();
  return (int)(rows < most ? (rows > 0 ? rows : 1) : most);
}

template <typename T>
int launch_norm_bwd(const T* g, const int8_t* codes, const uint8_t* exps, const float* w, const float* rms, T* gx,
                    float* gw, int64_t rows, int64_t cols, float* part, cudaStream_t st) {
  const bool vec = vec_ok<T>(g, cols, cols) && vec_ok<T>(gx, cols, cols) && vec_ok<float>(w, cols, cols);
  const RowPlan pl = row_plan(cols, vec);
  const int64_t pitch = ck_pitch(cols);
  const int blocks = norm_bwd_blocks(rows, cols);
  {
    ProfScope p("rmsnorm_checkpoint8_bwd", st);
#define MHC_NORM_BWD(VV, UU) \
  norm_bwd_kernel<T, VV, UU><<<blocks, pl.threads, 0, st>>>(g, codes, exps, w, rms, gx, part, rows, cols, pitch)
    if (pl.UPT == 0)
      norm_bwd_long_kernel<T><<<blocks, pl.threads, 0, st>>>(g, codes, exps, w, rms, gx, part, rows, cols, pitch);
    else if (pl.V == 8 && pl.UPT == 1) MHC_NORM_BWD(8, 1);
    else if (pl.V == 8 && pl.UPT == 2) MHC_NORM_BWD(8, 2);
    else if (pl.V == 8) MHC_NORM_BWD(8, 4);
    else if (pl.UPT == 1) MHC_NORM_BWD(1, 1);
    else if (pl.UPT == 4) MHC_NORM_BWD(1, 4);
    else if (pl.UPT == 8) MHC_NORM_BWD(1, 8);
    else MHC_NORM_BWD(1, 16);
#undef MHC_NORM_BWD
    const int rc = check_launch("rmsnorm_checkpoint8_bwd");
    if (rc) return rc;
  }
  ProfScope p("rmsnorm_checkpoint8_gw", st);
  norm_gw_kernel<<<(unsigned)((cols + 31) / 32), 256, 0, st>>>(part, gw, blocks, cols);
  return check_launch("rmsnorm_checkpoint8_gw");
}

int check_size(const char* what, int64_t rows, int64_t cols) {
  MHC_REQUIRE(rows >= 0 && cols >= 1, MHC_ERR_INVALID_ARG, "%s: rows must be >= 0 and cols >= 1 (got %lld x %lld)",
              what, (long long)rows, (long long)cols);
  MHC_REQUIRE(cols <= (1ll << 30) && rows <= (1ll << 40) / ck_pitch(cols), MHC_ERR_UNSUPPORTED,
              "%s: %lld x %lld values are too many", what, (long long)rows, (long long)cols);
  return MHC_OK;
}

int check_kept(const char* what, const int8_t* codes, const uint8_t* exps) {
  MHC_REQUIRE(codes != nullptr && exps != nullptr, MHC_ERR_INVALID_ARG, "%s: codes and exponents must not be NULL",
              what);
  MHC_REQUIRE(aligned16(codes) && (reinterpret_cast<uintptr_t>(exps) & 3) == 0, MHC_ERR_ALIGNMENT,
              "%s: codes must be 16-byte and exponents 4-byte aligned", what);
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int64_t mhc_checkpoint8_pitch(int64_t cols) { return cols > 0 ? ck_pitch(cols) : 0; }

extern "C" int mhc_checkpoint8_pack(const void* x, int32_t x_bf16, int64_t row_stride, int8_t* codes, uint8_t* exponents,
                                    int64_t rows, int64_t cols, void* stream) {
  int rc = check_size("checkpoint8_pack", rows, cols);
  if (rc) return rc;
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(x);
  MHC_REQUIRE(row_stride >= cols || rows == 1, MHC_ERR_INVALID_ARG, "checkpoint8_pack: row_stride %lld < cols %lld",
              (long long)row_stride, (long long)cols);
  rc = check_kept("checkpoint8_pack", codes, exponents);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  return x_bf16 ? launch_pack((const __nv_bfloat16*)x, row_stride, codes, exponents, rows, cols, st)
                : launch_pack((const float*)x, row_stride, codes, exponents, rows, cols, st);
}

extern "C" int mhc_checkpoint8_unpack(const int8_t* codes, const uint8_t* exponents, void* out, int32_t out_bf16,
                                      int64_t rows, int64_t cols, void* stream) {
  int rc = check_size("checkpoint8_unpack", rows, cols);
  if (rc) return rc;
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(out);
  rc = check_kept("checkpoint8_unpack", codes, exponents);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  return out_bf16 ? launch_unpack(codes, exponents, (__nv_bfloat16*)out, rows, cols, st)
                  : launch_unpack(codes, exponents, (float*)out, rows, cols, st);
}

extern "C" int mhc_rmsnorm_checkpoint8_fwd(const void* x, int32_t x_bf16, const float* weight, void* out, float* rms,
                                           int8_t* codes, uint8_t* exponents, int64_t rows, int64_t cols, float eps,
                                           void* stream) {
  int rc = check_size("rmsnorm_checkpoint8_fwd", rows, cols);
  if (rc) return rc;
  MHC_REQUIRE(eps >= 0.f, MHC_ERR_INVALID_ARG, "rmsnorm_checkpoint8_fwd: eps must be >= 0");
  MHC_REQUIRE(rows < (1ll << 31), MHC_ERR_UNSUPPORTED, "rmsnorm_checkpoint8_fwd: %lld rows are too many",
              (long long)rows);
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(x);
  MHC_REQUIRE_PTR(weight);
  MHC_REQUIRE_PTR(out);
  MHC_REQUIRE_PTR(rms);
  rc = check_kept("rmsnorm_checkpoint8_fwd", codes, exponents);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  return x_bf16 ? launch_norm_fwd((const __nv_bfloat16*)x, weight, (__nv_bfloat16*)out, rms, codes, exponents, rows,
                                  cols, eps, st)
                : launch_norm_fwd((const float*)x, weight, (float*)out, rms, codes, exponents, rows, cols, eps, st);
}

extern "C" size_t mhc_rmsnorm_checkpoint8_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1) return 0;
  return (size_t)norm_bwd_blocks(rows, cols) * (size_t)cols * sizeof(float);
}

extern "C" int mhc_rmsnorm_checkpoint8_bwd(const void* grad_out, int32_t g_bf16, const int8_t* codes,
                                           const uint8_t* exponents, const float* weight, const float* rms,
                                           void* grad_x, float* grad_weight, int64_t rows, int64_t cols,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_size("rmsnorm_checkpoint8_bwd", rows, cols);
  if (rc) return rc;
  MHC_REQUIRE_PTR(grad_weight);
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    cudaMemsetAsync(grad_weight, 0, (size_t)cols * sizeof(float), st);
    return check_launch("rmsnorm_checkpoint8_bwd");
  }
  MHC_REQUIRE_PTR(grad_out);
  MHC_REQUIRE_PTR(weight);
  MHC_REQUIRE_PTR(rms);
  MHC_REQUIRE_PTR(grad_x);
  rc = check_kept("rmsnorm_checkpoint8_bwd", codes, exponents);
  if (rc) return rc;
  MHC_REQUIRE(workspace != nullptr && workspace_bytes >= mhc_rmsnorm_checkpoint8_bwd_workspace_bytes(rows, cols),
              MHC_ERR_WORKSPACE, "rmsnorm_checkpoint8_bwd: workspace too small");
  float* part = (float*)workspace;
  return g_bf16 ? launch_norm_bwd((const __nv_bfloat16*)grad_out, codes, exponents, weight, rms, (__nv_bfloat16*)grad_x,
                                  grad_weight, rows, cols, part, st)
                : launch_norm_bwd((const float*)grad_out, codes, exponents, weight, rms, (float*)grad_x, grad_weight,
                                  rows, cols, part, st);
}
