// 8-bit activation checkpoints: pack, restore, and RMSNorm that keeps its
// input in 8 bits (forward and backward).  Format: checkpoint8.cuh.
#include "checkpoint8.cuh"
#include "tma.cuh"

namespace mhc {
namespace {

// ---------------------------------------------------------------------------
// pack / unpack: one pass, bound by HBM (a call among others, [32768, 4096] fp32:
// 97 and 104 us, 7.0 and 6.5 TB/s; [8192, 8192] bf16: 35 us each, 5.8 TB/s;
// uneven rows, [8192, 8191] fp32: 59 and 70 us, bf16: 84 and 66 us).  A warp takes
// spans of 256 columns of a row, a lane 8 of them (32 or 16 bytes in, 8 bytes of
// codes out), kUnroll spans at once so that enough loads are in flight.  EVEN:
// rows that 16- or 32-byte accesses fit; the spans then run over the rows without
// a gap.
// ---------------------------------------------------------------------------
constexpr int kPackThreads = 256, kUnroll = 4;

// Row and column of a lane's unit in a list of units, U (EVEN) or 32 * spans a row
// (64-bit divisions are a third of such a kernel's instructions: they are done in
// 32 bits, or not at all, wherever the numbers allow)
struct Walk {
  int64_t row, u, drow, du;
  __device__ __forceinline__ Walk(int64_t i, int64_t U) : row(0), u(i), drow(0), du(kPackThreads) {
    if (i >= U) {
      if ((uint64_t)i >> 32) {
        row = i / U;
        u = i - row * U;
      } else {
        row = (uint32_t)i / (uint32_t)U;
        u = (uint32_t)i % (uint32_t)U;
      }
    }
    if (U <= kPackThreads) {
      drow = kPackThreads / (int)U;
      du = kPackThreads % (int)U;
    }
  }
  __device__ __forceinline__ void step(int64_t U) {
    row += drow;
    u += du;
    if (u >= U) { u -= U; ++row; }
  }
};

// Rows without gaps and without padding: one list of units, and no index arithmetic
// (which is what bounds the general kernels in bf16: [8192, 8192] 54 us against 35).
template <typename T>
__global__ void __launch_bounds__(kPackThreads)
    pack_flat_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, uint8_t* __restrict__ exps, int64_t units) {
  const int64_t first = (int64_t)blockIdx.x * (kPackThreads * kUnroll) + threadIdx.x;
  x += 8 * first;
  codes += 8 * first;
  exps += first >> 2;
  const int left = (int)min((units - first + kPackThreads - 1) / kPackThreads, (int64_t)kUnroll);
  float v[kUnroll][8];
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
    if (k < left) ck_load(x + 8 * kPackThreads * k, v[k]);
  }
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) ck_encode(v[k], codes, exps, 8 * kPackThreads * k, k < left);
}
template <typename T>
__global__ void __launch_bounds__(kPackThreads)
    unpack_flat_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps, T* __restrict__ out,
                       int64_t units) {
  const int64_t first = (int64_t)blockIdx.x * (kPackThreads * kUnroll) + threadIdx.x;
  codes += 8 * first;
  exps += first >> 2;
  out += 8 * first;
  const int left = (int)min((units - first + kPackThreads - 1) / kPackThreads, (int64_t)kUnroll);
  uint2 w[kUnroll];
  uint32_t E[kUnroll];
#pragma unroll
  for (int k = 0; k < kUnroll; ++k)
    if (k < left) {
      w[k] = *reinterpret_cast<const uint2*>(codes + 8 * kPackThreads * k);
      E[k] = exps[kPackThreads / 4 * k];
    }
#pragma unroll
  for (int k = 0; k < kUnroll; ++k)
    if (k < left) {
      float v[8];
      ck_decode(w[k], E[k], v);
      ck_save(out + 8 * kPackThreads * k, v);
    }
}

template <typename T, bool EVEN>
__global__ void __launch_bounds__(kPackThreads)
    pack_kernel(const T* __restrict__ x, int64_t stride, int8_t* __restrict__ codes,
                uint8_t* __restrict__ exps, int64_t rows, int64_t cols, int64_t pitch, int64_t U) {
  __shared__ __align__(16) float sm[EVEN ? 1 : kPackThreads * 8];
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int64_t first = (int64_t)blockIdx.x * (kPackThreads * kUnroll) + threadIdx.x;
  Walk at(first, U);
  float v[kUnroll][8];
  int64_t row[kUnroll], col[kUnroll];
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    row[k] = at.row;
    col[k] = at.u * 8;
    if (EVEN) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
      if (at.row < rows && col[k] < cols) ck_load(x + at.row * stride + col[k], v[k]);  // cols % 8 == 0
    } else {  // U % 32 == 0: the warp is in one row
      ck_load_any(x + at.row * stride, col[k] - 8 * (threadIdx.x & 31), at.row < rows ? cols : 0, mine, v[k]);
    }
    at.step(U);
  }
#pragma unroll
  for (int k = 0; k < kUnroll; ++k)
    ck_encode(v[k], codes + row[k] * pitch, exps + row[k] * (pitch / kCkBlock), col[k], row[k] < rows && col[k] < pitch);
}

template <typename T, bool EVEN>
__global__ void __launch_bounds__(kPackThreads)
    unpack_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                  T* __restrict__ out, int64_t rows, int64_t cols, int64_t pitch, int64_t U) {
  __shared__ __align__(16) float sm[EVEN ? 1 : kPackThreads * 8];
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int64_t first = (int64_t)blockIdx.x * (kPackThreads * kUnroll) + threadIdx.x;
  Walk at(first, U);
  uint2 w[kUnroll];
  uint32_t E[kUnroll];
  int64_t row[kUnroll], col[kUnroll];
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    row[k] = at.row;
    col[k] = at.u * 8;
    w[k] = make_uint2(0u, 0u);
    E[k] = 1u;
    if (at.row < rows && col[k] < cols) {
      w[k] = *reinterpret_cast<const uint2*>(codes + at.row * pitch + col[k]);
      E[k] = exps[(at.row * pitch + col[k]) / kCkBlock];
    }
    at.step(U);
  }
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    float v[8];
    ck_decode(w[k], E[k], v);
    if (EVEN) {
      if (row[k] < rows && col[k] < cols) ck_save(out + row[k] * cols + col[k], v);
    } else {
      ck_save_any(out + row[k] * cols, col[k] - 8 * (threadIdx.x & 31), row[k] < rows ? cols : 0, mine, v);
    }
  }
}

// ---------------------------------------------------------------------------
// RMSNorm.  r = sqrt(mean x^2 + eps), y = x / r * w, and the codes of x, in one
// pass over x: a row stays in registers between the sum and the output, UPT
// units of 8 columns a thread.  WARP: rows of at most 1024 columns belong to a
// warp, 8 to a block, and need no barrier; longer ones to a block.
// ---------------------------------------------------------------------------
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

// Most threads of a block by the share of a row that one thread holds
constexpr int row_threads(int UPT, bool WARP) { return WARP || UPT == 1 ? 256 : UPT == 4 ? 1024 : 512; }

template <typename T, int UPT, bool WARP, bool EVEN>
__global__ void __launch_bounds__(row_threads(UPT, WARP))
    norm_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w, T* __restrict__ out,
                    float* __restrict__ rms, int8_t* __restrict__ codes, uint8_t* __restrict__ exps,
                    int64_t rows, int64_t cols, int64_t pitch, float eps) {
  __shared__ float red[32];
  extern __shared__ __align__(16) float sm[];  // uneven rows: 8 a thread
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int lane = threadIdx.x & 31;
  const int64_t row = WARP ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (WARP && row >= rows) return;
  const T* xr = x + row * cols;
  float v[UPT][8];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = unit_col<WARP>(k);
    if (EVEN) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
      if (c < cols) ck_load(xr + c, v[k]);
    } else {
      ck_load_any(xr, c - 8 * lane, cols, mine, v[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < UPT; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[k][j], v[k][j], ss);
  const float r = sqrtf(row_total<WARP>(ss, red) / (float)cols + eps), ir = 1.0f / r;
  if (WARP ? lane == 0 : threadIdx.x == 0) rms[row] = r;
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = unit_col<WARP>(k);
    float o[8], wv[8];
    load_w(w, c, cols, wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = v[k][j] * ir * wv[j];
    if (EVEN) {
      if (c < cols) ck_save(out + row * cols + c, o);
    } else {
      ck_save_any(out + row * cols, c - 8 * lane, cols, mine, o);
    }
    ck_encode(v[k], codes + row * pitch, exps + row * (pitch / kCkBlock), c, c < pitch);
  }
}

// Rows too long for registers: the row is read twice (the second time from L2).
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_fwd_long_kernel(const T* __restrict__ x, const float* __restrict__ w, T* __restrict__ out,
                         float* __restrict__ rms, int8_t* __restrict__ codes, uint8_t* __restrict__ exps,
                         int64_t cols, int64_t pitch, float eps) {
  __shared__ float red[32];
  __shared__ __align__(16) float sm[1024 * 8];
  float* mine = sm + (threadIdx.x >> 5) * 256;
  const int64_t row = blockIdx.x;
  const T* xr = x + row * cols;
  float ss = 0.f;
  for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
    const float t = ck_f32(xr[c]);
    ss = fmaf(t, t, ss);
  }
  const float r = sqrtf(row_total<false>(ss, red) / (float)cols + eps), ir = 1.0f / r;
  if (threadIdx.x == 0) rms[row] = r;
  for (int64_t c0 = (threadIdx.x >> 5) * 256; c0 < pitch; c0 += 8 * blockDim.x) {
    const int64_t c = c0 + 8 * (threadIdx.x & 31);
    float v[8], o[8], wv[8];
    ck_load_any(xr, c0, cols, mine, v);
    load_w(w, c, cols, wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = v[j] * ir * wv[j];
    ck_save_any(out + row * cols, c0, cols, mine, o);
    ck_encode(v, codes + row * pitch, exps + row * (pitch / kCkBlock), c, c < pitch);
  }
}

// Backward at the restored input xh:
//   gx = (g w - xh * D / (cols r^2)) / r,  D = sum_c g w xh
//   gw = sum over rows of g xh / r
// A block (or warp) walks every (its count)-th row; its threads keep their
// columns' share of gw in registers over all of them, so g and the codes are
// read once and gw leaves as one row of partial sums a block, added in block
// order by norm_gw_kernel: no atomics, the same bits every time.  The next
// row's g and codes are loaded before this row's sum is waited for.
// Uneven rows of a block are held to 64 registers, two blocks an SM: their loads
// wait on shared memory ([8192, 4097] bf16 by itself: 104 us against 186; among
// other calls, with the weight's sums, 112).
template <typename T, int UPT, bool WARP, bool EVEN>
__global__ void __launch_bounds__(row_threads(UPT, WARP), EVEN || WARP || UPT != 2 ? 1 : 2)
    norm_bwd_kernel(const T* __restrict__ g, const int8_t* __restrict__ codes,
                    const uint8_t* __restrict__ exps, const float* __restrict__ w,
                    const float* __restrict__ rms, T* __restrict__ gx, float* __restrict__ part,
                    int64_t rows, int64_t cols, int64_t pitch) {
  let_next_start();
  __shared__ float red[2][32];
  __shared__ __align__(16) float sm[EVEN && !WARP ? 1 : row_threads(UPT, WARP) * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* mine = sm + (EVEN ? 0 : warp * 256);
  float acc[UPT][8];
#pragma unroll
  for (int k = 0; k < UPT; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = 0.f;
  float ng[UPT][8];  // the row ahead
  uint2 nc[UPT];
  uint32_t ne[UPT];
  float nr = 1.f;
  auto fetch = [&](int64_t row) {
    if (row < rows) {
      nr = rms[row];
#pragma unroll
      for (int k = 0; k < UPT; ++k) {
        const int64_t c = unit_col<WARP>(k);
        nc[k] = make_uint2(0u, 0u);
        ne[k] = 1u;
        if (c < pitch) {
          nc[k] = *reinterpret_cast<const uint2*>(codes + row * pitch + c);
          ne[k] = exps[(row * pitch + c) / kCkBlock];
        }
        if (EVEN) {
#pragma unroll
          for (int j = 0; j < 8; ++j) ng[k][j] = 0.f;
          if (c < cols) ck_load(g + row * cols + c, ng[k]);
        } else {
          ck_load_any(g + row * cols, c - 8 * lane, cols, mine, ng[k]);
        }
      }
    }
  };
  const int64_t first = WARP ? (int64_t)blockIdx.x * kWarpRows + warp : (int64_t)blockIdx.x;
  const int64_t hop = WARP ? (int64_t)gridDim.x * kWarpRows : (int64_t)gridDim.x;
  fetch(first);
  int buf = 0;
  for (int64_t row = first; row < rows; row += hop, buf ^= 1) {
    float gv[UPT][8], xv[UPT][8];
    const float r = nr, ir = 1.0f / r;
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      float wv[8];
      load_w(w, unit_col<WARP>(k), cols, wv);
      ck_decode(nc[k], ne[k], xv[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[k][j] = fmaf(ng[k][j] * ir, xv[k][j], acc[k][j]);
        gv[k][j] = ng[k][j] * wv[j];
        d = fmaf(gv[k][j], xv[k][j], d);
      }
    }
    fetch(row + hop);
    // two buffers: a block writes red[buf] again only after the barrier of the row between
    const float coef = row_total<WARP>(d, red[buf]) / ((float)cols * r * r);
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int64_t c = unit_col<WARP>(k);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = (gv[k][j] - xv[k][j] * coef) * ir;
      if (EVEN) {
        if (c < cols) ck_save(gx + row * cols + c, o);
      } else {
        ck_save_any(gx + row * cols, c - 8 * lane, cols, mine, o);
      }
    }
  }
  if (WARP) {  // the warps' shares, added in warp order
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) sm[warp * 256 + j * 32 + lane] = acc[k][j];
      __syncthreads();
      float s = 0.f;
      for (int q = 0; q < kWarpRows; ++q) s += sm[q * 256 + threadIdx.x];
      const int64_t c = (k * 32 + lane) * 8 + (threadIdx.x >> 5);  // word j * 32 + lane holds column 8 lane + j
      if (c < cols) part[(int64_t)blockIdx.x * cols + c] = s;
    }
  } else {
#pragma unroll
    for (int k = 0; k < UPT; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = unit_col<WARP>(k) + j;
        if (c < cols) part[(int64_t)blockIdx.x * cols + c] = acc[k][j];
      }
  }
}

// ---------------------------------------------------------------------------
// Backward of rows of 1025 to 8192 columns that 16-byte copies fit: a block walks
// its rows over a ring of them in shared memory filled by bulk copies, so that
// what is in flight depends neither on registers nor on where the block's threads
// are.  g and xh are read from there twice, for the sum and for the output, so
// little is live across the barrier and 1024 threads fit an SM.  The barrier of
// row i also says that everyone is done with row i - 1: thread 0 then refills its
// place.  What bounds it is instructions (two expansions a value), hence two-wide
// fp32 arithmetic and the weights in shared memory.
// Measured at [16384, 7168] bf16: by itself 126 us, 4.7 TB/s (one row ahead in
// registers, a block an SM: 203 us); among other calls, with the weight's sums, 137
// us, [8192, 4096] bf16 58 us, fp32 72 us.
// ---------------------------------------------------------------------------
constexpr int kRingMost = 8, kRingUPT = 2;
constexpr int kRingBytes = 224 * 1024;  // of an SM's blocks together, two at least

struct Ring {
  int stages, blocks;  // blocks an SM; stages = 0: no ring
  uint32_t stage;      // bytes
  int threads;
};

// values of a unit in shared memory
__device__ __forceinline__ void smem_load(const float* p, float2 (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w);
  v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
}
__device__ __forceinline__ void smem_load(const __nv_bfloat16* p, float2 (&v)[4]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = make_float2(__uint_as_float(r[j] << 16), __uint_as_float(r[j] & 0xffff0000u));
}

template <typename T>
__global__ void __launch_bounds__(512, 2)
    norm_bwd_ring_kernel(const T* __restrict__ g, const int8_t* __restrict__ codes,
                         const uint8_t* __restrict__ exps, const float* __restrict__ w,
                         const float* __restrict__ rms, T* __restrict__ gx, float* __restrict__ part,
                         int64_t rows, int cols, int pitch, Ring plan) {
  let_next_start();
  extern __shared__ __align__(128) unsigned char ring_sm[];
  __shared__ uint64_t full[kRingMost];
  __shared__ float red[2][16];
  __shared__ int stop_s;
  volatile int* stop = &stop_s;
  constexpr int UPT = kRingUPT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const uint32_t gb = (uint32_t)cols * sizeof(T);  // bytes of a row of g; its codes follow
  float* ws = reinterpret_cast<float*>(ring_sm + (uint32_t)plan.stages * plan.stage);
  auto load = [&](int i, int s) {  // the block's row i into stage s; one thread
    const int64_t row = (int64_t)blockIdx.x + (int64_t)i * gridDim.x;
    if (row >= rows) return;
    unsigned char* dst = ring_sm + (uint32_t)s * plan.stage;
    mbar_expect_tx(&full[s], gb + (uint32_t)pitch);
    bulk_load(dst, g + row * cols, gb, &full[s]);
    bulk_load(dst + gb, codes + row * pitch, (uint32_t)pitch, &full[s]);
  };
  if (tid == 0) {
    for (int s = 0; s < plan.stages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    *stop = 0;
  }
  // The weights' first and second halves of units apart, so that eight lanes read
  // 128 bytes in a row: whole units met every bank twice (LSU 72% busy, 133 us
  // against 126 at [16384, 7168] bf16, by itself).
  const int units = cols / 8;
  for (int c = tid; c < cols; c += blockDim.x) ws[(((c >> 2) & 1) * units + (c >> 3)) * 4 + (c & 3)] = w[c];
  auto weights = [&](int c, float2 (&v)[4]) {
    const float4 a = reinterpret_cast<const float4*>(ws)[c >> 3], b = reinterpret_cast<const float4*>(ws)[units + (c >> 3)];
    v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w);
    v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
  };
  __syncthreads();
  if (tid == 0)
    for (int s = 0; s < plan.stages; ++s) load(s, s);
  int c[UPT];
  bool on[UPT];
  float2 acc[UPT][4];
  const uint8_t* ep = exps + (int64_t)blockIdx.x * (pitch / kCkBlock);
  uint32_t ne[UPT];  // the exponents and r of the row ahead
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    c[k] = 8 * (k * (int)blockDim.x + tid);
    on[k] = c[k] < cols;
    ne[k] = on[k] ? ep[c[k] / kCkBlock] : 1u;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[k][j] = make_float2(0.f, 0.f);
  }
  float nr = rms[blockIdx.x];
  const float share = 1.0f / (float)cols;
  int i = 0, s = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, ++i) {
    const unsigned char* at = ring_sm + (uint32_t)s * plan.stage;
    if (!mbar_wait(&full[s], phase)) *stop = 1;
    uint32_t E[UPT];
    const float ir = 1.0f / nr;
    float2 d2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      E[k] = ne[k];
      if (on[k]) {
        float2 gv[4], wv[4];
        float xv[8];
        smem_load(reinterpret_cast<const T*>(at) + c[k], gv);
        weights(c[k], wv);
        ck_decode(*reinterpret_cast<const uint2*>(at + gb + c[k]), E[k], xv);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 gx2 = __fmul2_rn(gv[j], make_float2(xv[2 * j], xv[2 * j + 1]));
          acc[k][j] = __ffma2_rn(gx2, make_float2(ir, ir), acc[k][j]);
          d2 = __ffma2_rn(gx2, wv[j], d2);
        }
      }
    }
    if (row + gridDim.x < rows) {
      ep += (int64_t)gridDim.x * (pitch / kCkBlock);
      nr = rms[row + gridDim.x];
#pragma unroll
      for (int k = 0; k < UPT; ++k)
        if (on[k]) ne[k] = ep[c[k] / kCkBlock];
    }
    const float d = warp_sum(d2.x + d2.y);
    if (lane == 0) red[i & 1][warp] = d;
    __syncthreads();
    if (*stop) break;
    if (tid == 0 && i > 0) load(i - 1 + plan.stages, s == 0 ? plan.stages - 1 : s - 1);
    float t = lane < nw ? red[i & 1][lane & 15] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);  // 16 warps at most
    const float coef = -__shfl_sync(0xffffffffu, t, 0) * share * (ir * ir);
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      if (on[k]) {
        float2 gv[4], wv[4];
        float xv[8], o[8];
        smem_load(reinterpret_cast<const T*>(at) + c[k], gv);
        weights(c[k], wv);
        ck_decode(*reinterpret_cast<const uint2*>(at + gb + c[k]), E[k], xv);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 a = __ffma2_rn(make_float2(xv[2 * j], xv[2 * j + 1]), make_float2(coef, coef),
                                      __fmul2_rn(gv[j], wv[j]));
          const float2 b = __fmul2_rn(a, make_float2(ir, ir));
          o[2 * j] = b.x;
          o[2 * j + 1] = b.y;
        }
        ck_save(gx + row * cols + c[k], o);
      }
    }
    if (++s == plan.stages) { s = 0; phase ^= 1; }
  }
  if (*stop && tid == 0)  // nothing may land after the block is gone
    for (int k = i; k < i + plan.stages; ++k)
      if ((int64_t)blockIdx.x + (int64_t)k * gridDim.x < rows)
        mbar_wait(&full[k % plan.stages], (uint32_t)((k / plan.stages) & 1));
#pragma unroll
  for (int k = 0; k < UPT; ++k)
    if (on[k]) {
      float* p = part + (int64_t)blockIdx.x * cols + c[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[2 * j] = acc[k][j].x;
        p[2 * j + 1] = acc[k][j].y;
      }
    }
}

// Rows too long for that: g and the codes are read twice (the second time from
// L2), and the block's share of gw is kept in shared memory (KEEP) or, past
// kKeepCols columns, in its row of partial sums.
constexpr int kLongThreads = 512;
constexpr int64_t kKeepCols = 49152;  // 192 KB; a multiple of the rows' padding

template <typename T, bool EVEN, bool KEEP>
__global__ void __launch_bounds__(kLongThreads)
    norm_bwd_long_kernel(const T* __restrict__ g, const int8_t* __restrict__ codes,
                         const uint8_t* __restrict__ exps, const float* __restrict__ w,
                         const float* __restrict__ rms, T* __restrict__ gx, float* __restrict__ part,
                         int64_t rows, int64_t cols, int64_t pitch) {
  let_next_start();
  extern __shared__ __align__(16) float keep[];  // [8][units]: value j of unit u at j * units + u
  __shared__ float red[2][32];
  __shared__ __align__(16) float sm[EVEN ? 1 : kLongThreads * 8];
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int lane = threadIdx.x & 31;
  const int64_t units = pitch / 8;
  float* p = KEEP ? keep : part + (int64_t)blockIdx.x * cols;
  auto slot = [&](int64_t c, int j) -> int64_t { return KEEP ? j * units + c / 8 : c + j; };
  // each unit is always the same thread's
  for (int64_t c = 8 * threadIdx.x; c < cols; c += 8 * kLongThreads)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) p[slot(c, j)] = 0.f;
  auto unit = [&](const T* gr, const int8_t* cr, const uint8_t* er, int64_t c, float (&gv)[8], float (&xv)[8]) {
    uint2 q = make_uint2(0u, 0u);
    uint32_t E = 1u;
    if (c < pitch) {
      q = *reinterpret_cast<const uint2*>(cr + c);
      E = er[c / kCkBlock];
    }
    ck_decode(q, E, xv);
    if (EVEN) {
#pragma unroll
      for (int j = 0; j < 8; ++j) gv[j] = 0.f;
      if (c < cols) ck_load(gr + c, gv);
    } else {
      ck_load_any(gr, c - 8 * lane, cols, mine, gv);
    }
  };
  int buf = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, buf ^= 1) {
    const int8_t* cr = codes + row * pitch;
    const uint8_t* er = exps + row * (pitch / kCkBlock);
    const T* gr = g + row * cols;
    const float r = rms[row], ir = 1.0f / r;
    float d = 0.f;
    for (int64_t c0 = 8 * (threadIdx.x & ~31); c0 < cols; c0 += 8 * kLongThreads) {
      const int64_t c = c0 + 8 * lane;
      float gv[8], xv[8], wv[8];
      unit(gr, cr, er, c, gv, xv);
      load_w(w, c, cols, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c + j < cols) p[slot(c, j)] = fmaf(gv[j] * ir, xv[j], p[slot(c, j)]);
        d = fmaf(gv[j] * wv[j], xv[j], d);
      }
    }
    const float coef = row_total<false>(d, red[buf]) / ((float)cols * r * r);
    for (int64_t c0 = 8 * (threadIdx.x & ~31); c0 < cols; c0 += 8 * kLongThreads) {
      const int64_t c = c0 + 8 * lane;
      float gv[8], xv[8], wv[8];
      unit(gr, cr, er, c, gv, xv);
      load_w(w, c, cols, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) gv[j] = (gv[j] * wv[j] - xv[j] * coef) * ir;
      if (EVEN) {
        if (c < cols) ck_save(gx + row * cols + c, gv);
      } else {
        ck_save_any(gx + row * cols, c0, cols, mine, gv);
      }
    }
  }
  if (KEEP)
    for (int64_t c = 8 * threadIdx.x; c < cols; c += 8 * kLongThreads)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < cols) part[(int64_t)blockIdx.x * cols + c + j] = p[slot(c, j)];
}

// gw[c] = sum of part[0..blocks)[c]: 32 columns a block, 8 threads a column,
// each a fixed share of the partial rows.
__global__ void __launch_bounds__(256)
    norm_gw_kernel(const float* __restrict__ part, float* __restrict__ gw, int blocks, int64_t cols) {
  __shared__ float s[8][32];
  wait_for_previous();
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

// How a row is laid over threads: UPT units a thread, `threads` a block; warp:
// one row a warp; UPT = 0: the row does not fit the registers.
struct RowPlan {
  int UPT, threads;
  bool warp;
};
RowPlan row_plan(int64_t cols, bool backward) {
  const int64_t pitch = ck_pitch(cols), U = pitch / 8;
  if (pitch <= kWarpCols) return {pitch <= 256 ? 1 : pitch <= 512 ? 2 : 4, 32 * kWarpRows, true};
  // forward: four units a thread wherever that leaves four warps, since small
  // blocks put more rows on an SM ([16384, 7168] bf16 by itself: 105 us against 118;
  // among other calls 110, 5.4 TB/s)
  if (!backward && U >= 512 && U <= 4096) return {4, (int)(((U + 3) / 4 + 31) / 32 * 32), false};
  for (int upt : {1, 2, 4}) {
    const int64_t th = (((U + upt - 1) / upt) + 31) / 32 * 32;
    if (th <= row_threads(upt, false)) return {upt, (int)th, false};
  }
  return {0, 1024, false};
}

template <typename T>
bool even_rows(const void* p, int64_t cols, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & (8 * sizeof(T) - 1)) == 0 && cols % 8 == 0 && stride % 8 == 0;
}

// Units of a row in pack's and unpack's list, and the list's blocks
int64_t list_units(int64_t cols, bool even, bool padded) {
  const int64_t u = ((padded ? ck_pitch(cols) : cols) + 7) / 8;
  return even ? u : (u + 31) / 32 * 32;
}
int64_t list_blocks(int64_t rows, int64_t U) {
  return (rows * U + kPackThreads * kUnroll - 1) / (kPackThreads * kUnroll);
}

template <typename T>
int launch_pack(const T* x, int64_t stride, int8_t* codes, uint8_t* exps, int64_t rows, int64_t cols,
                cudaStream_t st) {
  const bool even = even_rows<T>(x, cols, stride);
  const int64_t U = list_units(cols, even, true), blocks = list_blocks(rows, U), pitch = ck_pitch(cols);
  MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "checkpoint8_pack: %lld x %lld values are too many",
              (long long)rows, (long long)cols);
  ProfScope p("checkpoint8_pack", st);
  if (even && stride == cols && cols == pitch)
    pack_flat_kernel<T><<<(unsigned)blocks, kPackThreads, 0, st>>>(x, codes, exps, rows * U);
  else if (even) pack_kernel<T, true><<<(unsigned)blocks, kPackThreads, 0, st>>>(x, stride, codes, exps, rows, cols, pitch, U);
  else pack_kernel<T, false><<<(unsigned)blocks, kPackThreads, 0, st>>>(x, stride, codes, exps, rows, cols, pitch, U);
  return check_launch("checkpoint8_pack");
}

template <typename T>
int launch_unpack(const int8_t* codes, const uint8_t* exps, T* out, int64_t rows, int64_t cols, cudaStream_t st) {
  const bool even = even_rows<T>(out, cols, cols);
  const int64_t U = list_units(cols, even, false), blocks = list_blocks(rows, U), pitch = ck_pitch(cols);
  MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "checkpoint8_unpack: %lld x %lld values are too many",
              (long long)rows, (long long)cols);
  ProfScope p("checkpoint8_unpack", st);
  if (even && cols == pitch)
    unpack_flat_kernel<T><<<(unsigned)blocks, kPackThreads, 0, st>>>(codes, exps, out, rows * U);
  else if (even) unpack_kernel<T, true><<<(unsigned)blocks, kPackThreads, 0, st>>>(codes, exps, out, rows, cols, pitch, U);
  else unpack_kernel<T, false><<<(unsigned)blocks, kPackThreads, 0, st>>>(codes, exps, out, rows, cols, pitch, U);
  return check_launch("checkpoint8_unpack");
}

// LAUNCH(kernel) with the variant of KERNEL that the plan asks for
#define MHC_ROW_VARIANTS(KERNEL, LAUNCH)                                                                 \
  if (pl.warp) {                                                           \
    if (pl.UPT == 1) { if (even) LAUNCH((KERNEL<T, 1, true, true>)); else LAUNCH((KERNEL<T, 1, true, false>)); } \
    else if (pl.UPT == 2) { if (even) LAUNCH((KERNEL<T, 2, true, true>)); else LAUNCH((KERNEL<T, 2, true, false>)); } \
    else { if (even) LAUNCH((KERNEL<T, 4, true, true>)); else LAUNCH((KERNEL<T, 4, true, false>)); }       \
  } else if (pl.UPT == 1) { if (even) LAUNCH((KERNEL<T, 1, false, true>)); else LAUNCH((KERNEL<T, 1, false, false>)); } \
  else { if (even) LAUNCH((KERNEL<T, 2, false, true>)); else LAUNCH((KERNEL<T, 2, false, false>)); }

template <typename T>
int launch_norm_fwd(const T* x, const float* w, T* out, float* rms, int8_t* codes, uint8_t* exps, int64_t rows,
                    int64_t cols, float eps, cudaStream_t st) {
  const bool even = even_rows<T>(x, cols, cols) && even_rows<T>(out, cols, cols);
  const RowPlan pl = row_plan(cols, false);
  const int64_t pitch = ck_pitch(cols);
  const unsigned blocks = (unsigned)(pl.warp ? (rows + kWarpRows - 1) / kWarpRows : rows);
  ProfScope p("rmsnorm_checkpoint8_fwd", st);
  const size_t staging = even ? 0 : (size_t)pl.threads * 32;
#define MHC_NORM_FWD(KERN) KERN<<<blocks, pl.threads, staging, st>>>(x, w, out, rms, codes, exps, rows, cols, pitch, eps)
  if (pl.UPT == 0) {
    norm_fwd_long_kernel<T><<<blocks, pl.threads, 0, st>>>(x, w, out, rms, codes, exps, cols, pitch, eps);
  } else if (!pl.warp && pl.UPT == 4) {
    if (even) MHC_NORM_FWD((norm_fwd_kernel<T, 4, false, true>));
    else MHC_NORM_FWD((norm_fwd_kernel<T, 4, false, false>));
  } else {
    MHC_ROW_VARIANTS(norm_fwd_kernel, MHC_NORM_FWD)
  }
#undef MHC_NORM_FWD
  return check_launch("rmsnorm_checkpoint8_fwd");
}

// Rows whose backward does not fit the registers
bool long_bwd(const RowPlan& pl) { return !pl.warp && (pl.UPT == 0 || pl.UPT == 4); }

// Two to six blocks an SM, 1024 threads or less; the ring takes what the weights
// leave of 224 KB.
Ring ring_plan(int64_t rows, int64_t cols, size_t e) {
  const int64_t U = (cols + 7) / 8;
  Ring p = {0, 0, 0, 0};
  // a block has to meet several rows for its ring to pay
  if (ck_pitch(cols) <= kWarpCols || U > 1024 || rows < 8 * (int64_t)num_sms()) return p;
  p.threads = (int)((((U + kRingUPT - 1) / kRingUPT) + 31) / 32 * 32);
  p.blocks = 1024 / p.threads;
  p.blocks = p.blocks < 2 ? 2 : p.blocks > 6 ? 6 : p.blocks;
  p.stage = (uint32_t)((size_t)cols * e + ck_pitch(cols));
  const size_t s = ((size_t)(kRingBytes / p.blocks) - (size_t)cols * sizeof(float)) / p.stage;
  p.stages = (int)(s > kRingMost ? kRingMost : s);
  if (p.stages < 3) p.stages = 0;
  return p;
}

// Blocks of the backward: as many as run at once (the gradient of the weight
// leaves as one row a block), no more than there are rows for.
int norm_bwd_blocks(int64_t rows, int64_t cols) {
  const RowPlan pl = row_plan(cols, true);
  const Ring ring = ring_plan(rows, cols, 2);  // the blocks are the same for both types
  const int64_t need = pl.warp ? (rows + kWarpRows - 1) / kWarpRows : rows;
  const int64_t most = (ring.stages > 0 ? ring.blocks : 2) * (int64_t)num_sms();
  return (int)(need < most ? (need > 0 ? need : 1) : most);
}

template <typename T>
int launch_norm_bwd(const T* g, const int8_t* codes, const uint8_t* exps, const float* w, const float* rms, T* gx,
                    float* gw, int64_t rows, int64_t cols, float* part, cudaStream_t st) {
  const bool even = even_rows<T>(g, cols, cols) && even_rows<T>(gx, cols, cols);
  const RowPlan pl = row_plan(cols, true);
  const int64_t pitch = ck_pitch(cols);
  const int blocks = norm_bwd_blocks(rows, cols);
  {
    ProfScope p("rmsnorm_checkpoint8_bwd", st);
    const Ring ring = ring_plan(rows, cols, sizeof(T));
    // The limit on dynamic shared memory belongs to the kernel, not to the launch:
    // it is always set to the most that any width asks for, so that host threads
    // with other widths cannot lower it in between.
    if (even && ring.stages > 0) {
      auto kern = norm_bwd_ring_kernel<T>;
      const size_t bytes = (size_t)ring.stages * ring.stage + (size_t)cols * sizeof(float);
      constexpr int most = kRingBytes / 2;
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
        return fail(MHC_ERR_CUDA, "rmsnorm_checkpoint8_bwd: cannot reserve %d bytes of shared memory", most);
      kern<<<blocks, ring.threads, bytes, st>>>(g, codes, exps, w, rms, gx, part, rows, (int)cols, (int)pitch, ring);
    } else
#define MHC_NORM_BWD(KERN) KERN<<<blocks, pl.threads, 0, st>>>(g, codes, exps, w, rms, gx, part, rows, cols, pitch)
    if (long_bwd(pl)) {
      const bool keep = cols <= kKeepCols;
      const size_t bytes = keep ? (size_t)pitch * sizeof(float) : 0;
      auto go = [&](auto kern) -> int {
        constexpr int most = (int)(kKeepCols * sizeof(float));
        if (bytes && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
          return fail(MHC_ERR_CUDA, "rmsnorm_checkpoint8_bwd: cannot reserve %d bytes of shared memory", most);
        kern<<<blocks, kLongThreads, bytes, st>>>(g, codes, exps, w, rms, gx, part, rows, cols, pitch);
        return MHC_OK;
      };
      const int rc = keep ? (even ? go(norm_bwd_long_kernel<T, true, true>) : go(norm_bwd_long_kernel<T, false, true>))
                          : (even ? go(norm_bwd_long_kernel<T, true, false>) : go(norm_bwd_long_kernel<T, false, false>));
      if (rc) return rc;
    } else {
      MHC_ROW_VARIANTS(norm_bwd_kernel, MHC_NORM_BWD)
    }
#undef MHC_NORM_BWD
    const int rc = check_launch("rmsnorm_checkpoint8_bwd");
    if (rc) return rc;
  }
  ProfScope p("rmsnorm_checkpoint8_gw", st);
  launch_early(norm_gw_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(256), 0, st, part, gw, blocks, cols);
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

int norm_device_error(int* value, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_mhc_device_error, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && reset) e = cudaMemcpyToSymbol(g_mhc_device_error, &zero, sizeof(int));
  return e == cudaSuccess ? MHC_OK : fail(MHC_ERR_CUDA, "mhc_device_error_word: %s", cudaGetErrorString(e));
}

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
